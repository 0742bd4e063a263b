"""The 8-bit paged cache without a GPU: refusals of the C entry points and wrappers, struct layouts, the
workspace's size, and the 64-bit oracle's rounding against torch's fp8 conversion."""
import ctypes as C
import math

import pytest
import torch

from oracle import kv8_oracle as k8
from test_capi_exports import _c_struct_fields


@pytest.mark.parametrize("cname,pyname", [("mskv_kv8_pages", "Kv8PagesDesc"), ("mskv_kv8_append_desc", "Kv8AppendDesc"),
                                          ("mskv_kv8_score_desc", "Kv8ScoreDesc"), ("mskv_kv8_attn_desc", "Kv8AttnDesc")])
def test_struct_field_order(cname, pyname):
    from mserve_b200 import _lib
    assert [f[0] for f in getattr(_lib, pyname)._fields_] == _c_struct_fields(cname)


def _pages(d, **kw):
    """A valid description with addresses that nothing dereferences."""
    from mserve_b200 import _lib
    p = d.pages
    p.k, p.v, p.exps, p.bounds, p.page_table = 1 << 20, 2 << 20, 3 << 20, 4 << 20, 5 << 20
    p.stride_page, p.stride_h, p.pt_stride_b, p.num_pages = 2 * 16 * 128, 16 * 128, 8, 16
    p.max_pages, p.page_size, p.kv_heads, p.head_dim, p.dtype, p.batch = 8, 16, 2, 128, _lib.DT_FP8_E4M3, 2
    for name, value in kw.items():
        setattr(p, name, value)
    return d


def _append(**kw):
    from mserve_b200 import _lib
    d = _pages(_lib.Kv8AppendDesc())
    d.k_new, d.v_new, d.tok0, d.dtype, d.num_tokens = 6 << 20, 7 << 20, 8 << 20, _lib.DT_BF16, 3
    return d


def _score():
    from mserve_b200 import _lib
    d = _pages(_lib.Kv8ScoreDesc())
    d.q, d.lens, d.scores, d.scores_stride, d.dtype, d.q_heads, d.max_blocks = 6 << 20, 7 << 20, 8 << 20, 8, _lib.DT_F16, 14, 8
    return d


def _attn():
    from mserve_b200 import _lib
    d = _pages(_lib.Kv8AttnDesc())
    d.q, d.out, d.lens, d.workspace, d.workspace_bytes = 6 << 20, 7 << 20, 8 << 20, 9 << 20, 1 << 30
    d.scale, d.dtype, d.q_heads, d.q_len, d.max_tokens = 0.1, _lib.DT_BF16, 14, 1, 128
    return d


BAD_PAGES = [("k", None, "ARG"), ("exps", None, "ARG"), ("page_table", None, "ARG"), ("dtype", 1, "DTYPE"), ("batch", 0, "ARG"),
             ("kv_heads", -1, "ARG"), ("num_pages", 0, "ARG"), ("max_pages", 0, "ARG"), ("page_size", 8, "RANGE"),
             ("page_size", 24, "RANGE"), ("page_size", 256, "RANGE"), ("page_size", 0, "RANGE"), ("head_dim", 96, "RANGE"),
             ("k", (1 << 20) + 8, "ARG"), ("bounds", (4 << 20) + 4, "ARG"), ("stride_h", 2049, "ARG"), ("exps", 3, "ARG"),
             ("batch", 2 ** 30, "RANGE")]


@pytest.mark.parametrize("field,value,code", BAD_PAGES)
def test_c_refusals_of_the_cache(built_lib, field, value, code):
    from mserve_b200 import _lib
    lib = _lib.lib()
    for make, fn in ((_append, lib.mskv_kv8_append), (_score, lib.mskv_kv8_block_score), (_attn, lib.mskv_kv8_attention)):
        d = make()
        setattr(d.pages, field, value)
        assert fn(C.byref(d), None) == getattr(_lib, "MSKV_ERR_" + code), fn
        assert lib.mskv_last_error()


def test_c_refusals_of_the_calls(built_lib):
    from mserve_b200 import _lib
    lib = _lib.lib()
    for fn in (lib.mskv_kv8_append, lib.mskv_kv8_block_score, lib.mskv_kv8_attention):
        assert fn(None, None) == _lib.MSKV_ERR_ARG
    cases = [(_append, "mskv_kv8_append", [("dtype", _lib.DT_F64, "DTYPE"), ("num_tokens", -1, "ARG"), ("k_new", None, "ARG"),
                                           ("v_new", None, "ARG"), ("tok0", None, "ARG"), ("k_stride_t", 255, "ARG"),
                                           ("v_new", (7 << 20) + 1, "ARG")]),
             (_score, "mskv_kv8_block_score", [("dtype", _lib.DT_F32, "DTYPE"), ("q", None, "ARG"), ("lens", None, "ARG"),
                                               ("scores", None, "ARG"), ("q_heads", 13, "ARG"), ("q_heads", 0, "ARG"),
                                               ("max_blocks", 9, "ARG"), ("max_blocks", -1, "ARG"), ("scores_stride", 7, "ARG"),
                                               ("q_stride_h", 3, "ARG")]),
             (_attn, "mskv_kv8_attention", [("dtype", _lib.DT_F32, "DTYPE"), ("q", None, "ARG"), ("out", None, "ARG"),
                                            ("lens", None, "ARG"), ("q_heads", 13, "ARG"), ("q_heads", -2, "ARG"),
                                            ("q_len", 0, "RANGE"), ("q_len", 17, "RANGE"), ("max_tokens", 129, "ARG"),
                                            ("max_tokens", -1, "ARG"), ("scale", math.inf, "ARG"), ("scale", math.nan, "ARG"),
                                            ("out_stride_q", 1, "ARG")])]
    for make, name, bad in cases:
        for field, value, code in bad:
            d = make()
            setattr(d, field, value)
            assert getattr(lib, name)(C.byref(d), None) == getattr(_lib, "MSKV_ERR_" + code), (name, field, value)
    d = _score()
    d.pages.bounds = None
    assert lib.mskv_kv8_block_score(C.byref(d), None) == _lib.MSKV_ERR_ARG
    assert b"bounds" in lib.mskv_last_error()
    d = _attn()
    d.blocks, d.num_blocks = 10 << 20, -1
    assert lib.mskv_kv8_attention(C.byref(d), None) == _lib.MSKV_ERR_RANGE
    # nothing to append, nothing to score: done without a launch
    d = _append()
    d.num_tokens = 0
    assert lib.mskv_kv8_append(C.byref(d), None) == _lib.MSKV_OK
    d = _score()
    d.max_blocks = 0
    assert lib.mskv_kv8_block_score(C.byref(d), None) == _lib.MSKV_OK


def test_workspace(built_lib):
    """Long caches need a workspace and refuse a short or unaligned one; an invalid description needs 0 bytes."""
    from mserve_b200 import _lib
    lib = _lib.lib()
    d = _attn()
    d.pages.max_pages, d.max_tokens = 1 << 16, 1 << 20
    need = lib.mskv_kv8_attention_workspace_bytes(C.byref(d))
    assert need > 0
    for field, value in (("workspace_bytes", need - 1), ("workspace", None), ("workspace", (9 << 20) + 4)):
        bad = _attn()
        bad.pages.max_pages, bad.max_tokens, bad.workspace_bytes = 1 << 16, 1 << 20, need
        setattr(bad, field, value)
        assert lib.mskv_kv8_attention(C.byref(bad), None) == _lib.MSKV_ERR_ARG
        assert b"workspace" in lib.mskv_last_error()
    d.q_len = 99
    assert lib.mskv_kv8_attention_workspace_bytes(C.byref(d)) == 0


@pytest.fixture(scope="session")
def ext(built_lib):
    from mserve_b200 import build
    return build.build_kv8_ext()


def test_new_pages(built_lib):
    from mserve_b200 import ops
    with pytest.raises(TypeError):
        ops.kv8_pages(4, 2, 128, dtype=torch.float16, device="cpu")
    for kw in ({"page_size": 8}, {"page_size": 144}, {"head_dim": 80}):
        with pytest.raises(ValueError):
            ops.kv8_pages(4, 2, **{"head_dim": 128, "device": "cpu", **kw})
    pages = ops.kv8_pages(4, 2, 128, device="cpu")
    assert pages.k.shape == (4, 2, 16, 128) and pages.bounds.shape == (4, 2, 2, 128) and pages.exps.dtype == torch.int8
    assert not pages.k.view(torch.uint8).any() and pages.k.data_ptr() != pages.v.data_ptr()
    assert ops.kv8_pages(4, 2, 64, device="cpu", bounds=False).bounds is None


def _calls(pages, table, B=1, D=128):
    """The three operators on CPU tensors; well-formed calls get as far as the device check."""
    from mserve_b200 import ops
    n = torch.zeros(B, dtype=torch.int32)
    x = torch.zeros(B, 2, 3, D, dtype=torch.bfloat16)
    q = torch.zeros(B, 6, 1, D, dtype=torch.bfloat16)
    return [lambda **kw: ops.kv8_append(**{**dict(pages=pages, page_table=table, k_new=x, v_new=x, tok0=n), **kw}),
            lambda **kw: ops.kv8_block_score(**{**dict(q=q, pages=pages, page_table=table, lens=n, max_blocks=1,
                                                       out=torch.zeros(B, 2, 1)), **kw}),
            lambda **kw: ops.kv8_attention(**{**dict(q=q, pages=pages, page_table=table, lens=n), **kw})]


def test_cpu_tensors_are_refused(ext):
    from mserve_b200 import ops
    pages, table = ops.kv8_pages(4, 2, 128, device="cpu"), torch.zeros(1, 5, dtype=torch.int32)
    for call in _calls(pages, table):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_the_cache_is_checked(ext):
    """Every tensor of the cache by shape, type and layout."""
    from mserve_b200 import ops
    pages, table = ops.kv8_pages(4, 2, 128, device="cpu"), torch.zeros(3, 5, dtype=torch.int32)
    u8 = lambda t: t.view(torch.uint8)  # noqa: E731
    bad = [pages._replace(k=u8(pages.k)), pages._replace(v=pages.v[:2]), pages._replace(v=pages.v.view(torch.float8_e5m2)),
           pages._replace(k=pages.k.transpose(2, 3)), pages._replace(exps=pages.exps[:3]), pages._replace(exps=u8(pages.exps)),
           pages._replace(exps=pages.exps[:, :1]), pages._replace(bounds=pages.bounds[..., :64]), pages._replace(bounds=u8(pages.bounds)),
           pages._replace(k=pages.k[:, :, :, ::2], v=pages.v[:, :, :, ::2]), pages._replace(k=pages.k[0], v=pages.v[0]),
           pages._replace(exps=pages.exps.transpose(0, 1).contiguous().transpose(0, 1))]
    for b in bad:
        for call in _calls(pages, table, B=3):
            with pytest.raises(ValueError, match="must"):
                call(pages=b)
    for t in (table.long(), table[:2], table.t(), table[0], torch.zeros(3, 10, dtype=torch.int32)[:, ::2]):
        for call in _calls(pages, table, B=3):
            with pytest.raises(ValueError, match="page_table"):
                call(page_table=t)


def test_the_arguments_are_checked(ext):
    from mserve_b200 import ops
    pages, table = ops.kv8_pages(4, 2, 128, device="cpu"), torch.zeros(1, 5, dtype=torch.int32)
    append, score, attend = _calls(pages, table)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    x = torch.zeros(1, 2, 3, 128, dtype=torch.bfloat16)
    for kw, error in [(dict(v_new=x[:, :, :2]), ValueError), (dict(v_new=x.half()), ValueError), (dict(k_new=x[0], v_new=x[0]), ValueError),
                      (dict(k_new=x[..., :64], v_new=x[..., :64]), ValueError), (dict(k_new=x[:, :1], v_new=x[:, :1]), ValueError),
                      (dict(k_new=x.int(), v_new=x.int()), TypeError), (dict(k_new=x.double(), v_new=x.double()), TypeError),
                      (dict(k_new=x.repeat(1, 1, 1, 2)[..., ::2], v_new=x), ValueError), (dict(tok0=i32(2)), ValueError),
                      (dict(tok0=torch.zeros(1)), ValueError), (dict(counts=i32(3)), ValueError)]:
        with pytest.raises(error):
            append(**kw)
    q = torch.zeros(1, 6, 1, 128, dtype=torch.bfloat16)
    for kw, error in [(dict(q=q.float()), TypeError), (dict(q=q[..., :64]), ValueError), (dict(q=q[:, :5]), ValueError),
                      (dict(q=q[0, 0]), ValueError), (dict(lens=i32(2)), ValueError), (dict(lens=torch.zeros(1)), ValueError),
                      (dict(q=q.repeat(1, 1, 1, 2)[..., ::2]), ValueError)]:
        for call in (score, attend):
            with pytest.raises(error):
                call(**kw)
    for kw in (dict(max_blocks=6, out=torch.zeros(1, 2, 9)), dict(max_blocks=-1), dict(max_blocks=2), dict(out=torch.zeros(1, 1, 4)),
               dict(out=torch.zeros(1, 2, 4).double()), dict(out=torch.zeros(1, 2, 8)[..., ::2]), dict(pages=pages._replace(bounds=None))):
        with pytest.raises(ValueError, match="max_blocks|out must|bounds"):
            score(**kw)
    for kw in (dict(max_tokens=81), dict(max_tokens=-1), dict(q=q.expand(1, 6, 17, 128)), dict(q=q[:, :, :0]), dict(scale=math.inf),
               dict(scale=math.nan), dict(blocks=i32(1, 2)), dict(blocks=i32(1, 1, 4)), dict(blocks=i32(1, 2, 4).long()),
               dict(blocks=i32(1, 2, 8)[..., ::2]), dict(counts=i32(1, 2)), dict(blocks=i32(1, 2, 4), counts=i32(1)),
               dict(out=torch.zeros_like(q).half()), dict(out=torch.zeros(1, 6, 2, 128, dtype=torch.bfloat16))):
        with pytest.raises(ValueError, match="must|counts go"):
            attend(**kw)


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.float8_e5m2])
def test_oracle_rounding(dtype):
    """The oracle's rounding is torch's (round to nearest even) wherever nothing saturates; every code is a fixed point."""
    codes = torch.arange(256, dtype=torch.uint8).view(dtype).double()
    finite = torch.isfinite(codes)
    assert torch.equal(k8.nearest_code(codes[finite], dtype), codes[finite])
    g = torch.Generator().manual_seed(0)
    x = torch.randn(20000, generator=g) * torch.exp2(torch.randint(-20, 8, (20000,), generator=g).float())
    x = x.clamp(-400, 400)
    assert torch.equal(k8.nearest_code(x.double(), dtype), x.to(dtype).double())
    half = (codes[finite].sort().values[1:] + codes[finite].sort().values[:-1]) / 2
    assert torch.equal(k8.nearest_code(half, dtype), half.float().to(dtype).double())
    assert float(k8.nearest_code(torch.tensor([math.inf], dtype=torch.float64), dtype)) == k8.F8[dtype][2]


def test_oracle_exponent():
    for dtype in k8.F8:
        top = k8.F8[dtype][2]
        for e in (-60, -3, 0, 1, 60):
            x = torch.tensor([top * 2.0 ** e, -1.0 * 2.0 ** -70], dtype=torch.float64)
            assert k8.page_exponent(x, dtype) == e
            assert k8.page_exponent(x * (1 + 2.0 ** -20), dtype) == min(e + 1, 60)
        assert k8.page_exponent(torch.tensor([math.nan, math.inf, 0.0], dtype=torch.float64), dtype) == -60
