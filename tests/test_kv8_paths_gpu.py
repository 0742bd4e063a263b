"""The 8-bit cache's kernels at the sizes that choose their other variants: appends of many pages, block scores of several
tiles a warp, attention whose work is one line cut across segments.  Each case asserts that it is of the variant.

Page tables name a page more than once where a case only reads: a long cache without its memory.
"""
import ctypes as C
import math

import pytest
import torch

from oracle import kv8_oracle as k8
from test_kv8_gpu import E4M3, E5M2, _bits, _close, _filled, _host, _i32, _same, _table

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


# ---- append: more than four pages of a KV head for every multiprocessor ---------------------------
def _rows(g, B, H, n, D, new, values, layout):
    """New rows: normal numbers of growing size along the tokens, some of them special; a view of the layout."""
    x = torch.randn(B, H, n, D, generator=g) * torch.exp2(torch.randint(-12, 10, (B, H, n, 1), generator=g).float())
    if values == "special":
        pick = torch.randint(0, 400, (B, H, n, 1), generator=g)       # some rows have one special element
        at = torch.arange(D) == torch.randint(0, D, (B, H, n, 1), generator=g)
        for i, s in enumerate([math.inf, -math.inf, math.nan, -math.nan, 0.0, 6e-8, -3e-39, 6e4]):
            x = torch.where((pick == i) & at, torch.tensor(s), x)
        x[:, 0, 16:40] = 0.0                                          # pages of zeros, of NaN, of infinities
        x[:, 1, 32:130] = math.nan
        x[0, :, 140:300] = math.inf
    x = x.to(new)
    if layout == "heads":
        return x.cuda()
    if layout == "tokens":                                            # as a fused projection leaves them
        return x.transpose(1, 2).contiguous().cuda().transpose(1, 2)
    buf = torch.zeros(B, n, H * D + 3, dtype=new, device="cuda")      # rows that start at odd elements
    v = buf[:, :, 1:1 + H * D].view(B, n, H, D).transpose(1, 2)
    v.copy_(x)
    assert v.data_ptr() % 16 and v.stride(2) % 8
    return v


@pytest.mark.parametrize("new,D,page,cache,values,layout", [
    (BF16, 128, 16, E4M3, "special", "heads"), (F16, 128, 16, E4M3, "special", "heads"), (BF16, 64, 16, E5M2, "special", "tokens"),
    (BF16, 256, 16, E4M3, "special", "odd"), (F16, 64, 32, E5M2, "special", "odd"), (F16, 256, 32, E4M3, "normal", "tokens"),
    (BF16, 128, 48, E4M3, "special", "heads"), (F16, 128, 64, E5M2, "special", "tokens"), (BF16, 64, 80, E4M3, "special", "odd"),
    (BF16, 128, 128, E4M3, "special", "heads"), (F16, 256, 128, E5M2, "special", "heads"), (BF16, 256, 64, E5M2, "special", "odd"),
    (F32, 128, 16, E4M3, "special", "heads"), (F32, 64, 32, E5M2, "special", "odd"), (F32, 256, 48, E4M3, "special", "tokens"),
    (F32, 128, 128, E5M2, "normal", "tokens")])
def test_append_of_many_pages(built_lib, new, D, page, cache, values, layout):
    """A prompt, ragged, then as many tokens again behind it: pages of new rows only, pages that join old ones, all in one
    launch of several pages a CTA; bit for bit."""
    from mserve_b200 import ops
    B, H = 5, 8
    n = page * (4 * _sms() // (B * H) + 2)
    touched = (n + page - 2) // page + 1
    assert touched * B * H > 4 * _sms()
    g = torch.Generator().manual_seed(D + page)
    width = 2 * touched + 1
    table = _table(B, width, 4, g)
    pages = ops.kv8_pages(B * width + 4, H, D, page_size=page, dtype=cache)
    want = _host(pages)
    tok0 = torch.zeros(B, dtype=torch.int32)
    for counts in ([n, n - 7, page + 1, 0, n - page], [n - 1, 1, n, n, 5]):
        k, v = (_rows(g, B, H, n, D, new, values, layout) for _ in range(2))
        cnt = torch.tensor(counts, dtype=torch.int32)
        ops.kv8_append(pages, table.cuda(), k, v, tok0=tok0.cuda(), counts=cnt.cuda())
        want = k8.append(want, table, k.cpu().double(), v.cpu().double(), tok0, cnt, cache)
        _same(pages, want)
        tok0 += cnt
    ops.check_status(torch.device("cuda"))


def test_append_of_many_pages_without_bounds(built_lib):
    """A cache that keeps no bounds, and K and V pools inside one allocation: nothing outside the written rows changes."""
    from mserve_b200 import ops
    B, H, D, page = 6, 7, 128, 16
    n = page * (4 * _sms() // (B * H) + 2) - 3
    width = n // page + 1
    g = torch.Generator().manual_seed(1)
    both = torch.randint(0, 120, (B * width + 2, 2, H, page, D), dtype=torch.uint8, generator=g).cuda().view(E4M3)
    pages = ops.Kv8Pages(both[:, 0], both[:, 1], torch.zeros(B * width + 2, H, 2, dtype=torch.int8, device="cuda"), None)
    table = _table(B, width, 2, g)
    k, v = (torch.randn(B, H, n, D, generator=g).to(BF16).cuda() for _ in range(2))
    start = {"k": pages.k.cpu().double(), "v": pages.v.cpu().double(), "exps": pages.exps.cpu().long(),
             "bounds": torch.zeros(B * width + 2, H, 2, D, dtype=torch.float64)}
    want = k8.append(start, table, k.cpu().double(), v.cpu().double(), [0] * B, [n] * B, E4M3)
    ops.kv8_append(pages, table.cuda(), k, v, tok0=torch.zeros(B, dtype=torch.int32, device="cuda"))
    ops.check_status(torch.device("cuda"))
    for name in ("k", "v", "exps"):
        assert torch.equal(getattr(pages, name).cpu().double(), want[name].double()), name


def test_append_of_many_pages_bad_destinations(built_lib):
    """Unmapped pages and tokens past the table among many good ones: skipped and reported, the others written."""
    from mserve_b200 import ops
    B, H, D, page = 4, 8, 64, 16
    width = 4 * _sms() // (B * H) + 3
    n = page * (width + 1)
    g = torch.Generator().manual_seed(2)
    table = _table(B, width, 0, g)
    bad = table.clone()
    bad[1, 3], bad[2, width - 1] = -1, B * width
    pages, good = (ops.kv8_pages(B * width, H, D, page_size=page) for _ in range(2))
    k, v = (torch.randn(B, H, n, D, generator=g).to(BF16).cuda() for _ in range(2))
    zero = torch.zeros(B, dtype=torch.int32, device="cuda")
    ops.kv8_append(good, table.cuda(), k, v, tok0=zero, counts=zero + page * width)
    ops.check_status(torch.device("cuda"))
    ops.kv8_append(pages, bad.cuda(), k, v, tok0=zero)
    with pytest.raises(RuntimeError, match="not mapped.*destination|destination.*not mapped"):
        ops.check_status(torch.device("cuda"))
    keep = torch.ones(B * width, dtype=torch.bool)
    keep[table[1, 3].long()] = keep[table[2, width - 1].long()] = False
    for a, b in zip(pages, good):
        a, b = a.view(torch.uint8).cpu(), b.view(torch.uint8).cpu()
        assert torch.equal(a[keep], b[keep]) and not a[~keep].any()


# ---- block scores: two to four tiles a warp -------------------------------------------------------
@pytest.mark.parametrize("D,page,cache,qt,G,tiles", [(64, 16, E4M3, BF16, 7, 2), (128, 16, E4M3, F16, 5, 3), (128, 32, E5M2, BF16, 1, 4),
                                                     (256, 16, E4M3, BF16, 2, 4), (64, 128, E5M2, F16, 12, 4), (256, 64, E5M2, F16, 3, 2)])
def test_block_scores_of_several_tiles(built_lib, D, page, cache, qt, G, tiles):
    from mserve_b200 import ops
    B, H, P = 8, 4, 700
    rows = -(-2 * _sms() * tiles // (B * H))
    nb = 128 * rows - 37
    assert min(4, B * H * rows // (2 * _sms())) == tiles
    g = torch.Generator().manual_seed(D + tiles)
    src, _, _ = _filled(1, H, D, page, cache, [P * page], seed=D, spare=0)     # P pages, named again and again
    table = torch.randint(0, P, (B, nb), generator=g).to(torch.int32)
    lens = [nb * page, nb * page - page // 2, 0, 1, 128 * tiles * page + 1, 127 * page, (nb - 128) * page, 5 * page]
    q = (torch.randn(B, H * G, D, generator=g) * torch.exp2(torch.randint(-9, 6, (1, 1, D), generator=g).float())).to(qt)
    out = torch.full((B, H, nb + 5), 7.0, device="cuda")
    ops.kv8_block_score(q.cuda(), src, table.cuda(), lens=_i32(lens), max_blocks=nb, out=out)
    ops.check_status(torch.device("cuda"))
    # the definition: each query head's largest product element by element; the same with magnitudes
    bounds, e = src.bounds.double(), torch.pow(2.0, src.exps[:, :, 0].double())
    at = table.long().cuda()
    qd = q.double().cuda().view(B, H, G, D)
    top = qd.abs().sum(dim=2).amax(dim=-1)
    got = out.double()
    for b in range(B):
        held = -(-lens[b] // page)
        assert (got[b, :, held:] == 7).all()
        for h in range(H):
            c = bounds[at[b, :held], h]                                          # [held, 2, D]
            s = e[at[b, :held], h]
            want = sum(torch.maximum(qd[b, h, i] * c[:, 0], qd[b, h, i] * c[:, 1]).sum(dim=-1) for i in range(G)) * s
            mag = sum((qd[b, h, i].abs() * c.abs().amax(dim=1)).sum(dim=-1) for i in range(G)) * s
            # 2D/16 + 4 roundings of 2^-22, the weights' 23 bits of the largest, the G terms of a weight
            tol = mag * (2 * D / 16 + 4) * 2.0 ** -22 + c.abs().sum(dim=(1, 2)) * s * top[b, h] * 2.0 ** -23 + G * mag * 2.0 ** -24
            off = (got[b, h, :held] - want).abs()
            assert (off <= tol).all(), (b, h, float((off / tol).max()))


def test_block_scores_of_several_tiles_bad_pages(built_lib):
    """Unmapped pages in the second tile and later: -inf there, the neighbours as without them."""
    from mserve_b200 import ops
    B, H, D, G, P, page = 8, 4, 64, 2, 50, 16
    rows = -(-2 * _sms() * 3 // (B * H))
    nb = 128 * rows
    g = torch.Generator().manual_seed(9)
    src, _, _ = _filled(1, H, D, page, E4M3, [P * page], seed=9, spare=0)
    table = torch.randint(0, P, (B, nb), generator=g).to(torch.int32)
    q = torch.randn(B, H * G, D, generator=g).to(BF16).cuda()
    lens = _i32([nb * page] * B)
    good, out = (torch.zeros(B, H, nb, device="cuda") for _ in range(2))
    ops.kv8_block_score(q, src, table.cuda(), lens=lens, max_blocks=nb, out=good)
    ops.check_status(torch.device("cuda"))
    bad = torch.zeros(B, nb, dtype=torch.bool)
    for j in (130, 255, 256, 300, nb - 1):
        bad[:, j] = True
    t = torch.where(bad, torch.where(torch.arange(nb) % 2 == 0, torch.tensor(-1), torch.tensor(src.k.shape[0])).to(torch.int32), table)
    ops.kv8_block_score(q, src, t.cuda(), lens=lens, max_blocks=nb, out=out)
    with pytest.raises(RuntimeError, match="not mapped"):
        ops.check_status(torch.device("cuda"))
    bad = bad.cuda()[:, None].expand(-1, H, -1)
    assert (out[bad] == -math.inf).all() and torch.equal(out[~bad], good[~bad])


# ---- attention: one line of tiles, its parts across segments -------------------------------------
def _line_ctas(B, H, G, D, Q, page, width, max_tokens, S=None):
    """CTAs of a call that goes by the line, from its workspace; 0 for one that needs none."""
    from mserve_b200 import _lib
    d = _lib.Kv8AttnDesc()
    p = d.pages
    p.k, p.v, p.exps, p.page_table = 1 << 20, 2 << 20, 3 << 20, 4 << 20
    p.stride_page, p.stride_h, p.pt_stride_b, p.num_pages = H * page * D, page * D, width, 1 << 20
    p.max_pages, p.page_size, p.kv_heads, p.head_dim, p.dtype, p.batch = width, page, H, D, _lib.DT_FP8_E4M3, B
    d.scale, d.dtype, d.q_heads, d.q_len, d.max_tokens = 0.1, _lib.DT_BF16, H * G, Q, max_tokens
    if S is not None:
        d.blocks, d.num_blocks = 5 << 20, S
    need = _lib.lib().mskv_kv8_attention_workspace_bytes(C.byref(d))
    if need == 0:
        return 0, 0
    nt = 1 if G * Q <= 8 or D == 256 else 2
    segments = B * H * -(-G * Q // (8 * nt))
    up = lambda x: -(-x // 256) * 256  # noqa: E731
    ctas = [c for c in range(1, 4096) if up(segments * 16) + up(c * nt * 128) + c * nt * 16 * D * 4 == need]
    assert len(ctas) == 1
    return ctas[0], segments


LINES = [  # B, H, G, D, Q, page, cache, query type, bound of the lengths, parts for each CTA that runs at once
    (50, 4, 7, 128, 1, 16, E4M3, BF16, 6000, 1), (80, 4, 7, 128, 1, 32, E5M2, F16, 8000, 2),
    (10, 3, 7, 128, 5, 16, E4M3, F16, 6000, 1), (20, 4, 14, 128, 4, 64, E5M2, BF16, 12000, 2),
    (10, 4, 5, 256, 5, 16, E4M3, BF16, 5000, 1), (90, 2, 3, 256, 1, 48, E5M2, F16, 9000, 2),
    (60, 4, 5, 64, 1, 16, E4M3, BF16, 12000, 1), (70, 8, 8, 64, 1, 128, E5M2, F16, 16000, 2),
    (45, 4, 12, 64, 1, 32, E4M3, F16, 6000, 1), (30, 4, 9, 64, 4, 16, E4M3, BF16, 9000, 2)]


def _at_once(D, rows):
    """CTAs that run at once."""
    return _sms() * (1 if D == 256 else 3 if D == 64 and rows <= 8 else 2 if D == 64 or rows <= 8 else 1)


def _ragged(B, most, g):
    lens = (40 * torch.rand(B, generator=g).mul(4).exp()).long().tolist()      # 40 to 2000, most of them short
    lens[0], lens[1], lens[3], lens[B // 2], lens[-2], lens[-1] = most, 0, 1, most // 2 + 3, 0, 17
    return lens


@pytest.mark.parametrize("B,H,G,D,Q,page,cache,qt,most,waves", LINES)
def test_line_across_segments(built_lib, B, H, G, D, Q, page, cache, qt, most, waves):
    """CTAs that end one segment and begin others, among them empty ones; segments of several CTAs, whole ones, several row
    tiles of one sequence."""
    from mserve_b200 import ops
    P, width = 90, -(-most // page)
    ctas, segments = _line_ctas(B, H, G, D, Q, page, width, most)
    assert ctas == waves * _at_once(D, G * Q) and segments * 2 > ctas
    g = torch.Generator().manual_seed(B + D + Q)
    pages, _, _ = _filled(1, H, D, page, cache, [P * page], seed=D + B, spare=0)
    table = torch.randint(0, P, (B, width), generator=g).to(torch.int32)
    lens = _ragged(B, most, g)
    q = (torch.randn(B, H * G, Q, D, generator=g) * 0.5).to(qt)
    out = torch.full(q.shape, float("nan"), dtype=qt, device="cuda")
    ops.kv8_attention(q.cuda(), pages, table.cuda(), lens=_i32(lens), max_tokens=most, out=out)
    ops.check_status(torch.device("cuda"))
    want, bound = k8.attention(q.double(), _host(pages), table, lens, weight_bits=_bits(qt))
    _close(out, want, bound)
    again = torch.full_like(out, float("nan"))
    ops.kv8_attention(q.cuda(), pages, table.cuda(), lens=_i32(lens), max_tokens=most, out=again)
    assert torch.equal(out, again)


@pytest.mark.parametrize("B,H,G,D,Q,page,cache,qt,most,waves", LINES[::2])
def test_line_across_segments_of_lists(built_lib, B, H, G, D, Q, page, cache, qt, most, waves):
    """The same over lists, whose units are (sequence, KV head): counts of zero, of one, of all; entries that repeat."""
    from mserve_b200 import ops
    P, S, width = 90, 640 // (page // 16), 200
    ctas, segments = _line_ctas(B, H, G, D, Q, page, width, width * page, S)
    assert ctas and segments * 2 > ctas
    g = torch.Generator().manual_seed(B + D + Q)
    pages, _, _ = _filled(1, H, D, page, cache, [P * page], seed=D + B, spare=0)
    table = torch.randint(0, P, (B, width), generator=g).to(torch.int32)
    lens = torch.randint(1, width * page, (B,), generator=g).tolist()
    lens[2] = 0
    counts = (torch.rand(B, H, generator=g) * 4.5).exp().int()                 # 1 to 90
    counts[0, 0], counts[1], counts[B // 2, 1], counts[B - 1, -1] = S, 0, S // 2, 0
    blocks = torch.full((B, H, S), 2 ** 30, dtype=torch.int32)
    for b in range(B):
        held = max(-(-lens[b] // page), 1)
        for h in range(H):
            blocks[b, h, :counts[b, h]] = torch.randint(0, held, (int(counts[b, h]),), generator=g).int()
    q = (torch.randn(B, H * G, Q, D, generator=g) * 0.5).to(qt)
    out = torch.full(q.shape, float("nan"), dtype=qt, device="cuda")
    ops.kv8_attention(q.cuda(), pages, table.cuda(), lens=_i32(lens), blocks=blocks.cuda(), counts=counts.cuda(), out=out)
    ops.check_status(torch.device("cuda"))
    want, bound = k8.attention(q.double(), _host(pages), table, lens, blocks=blocks, counts=counts, weight_bits=_bits(qt))
    _close(out, want, bound)


@pytest.mark.parametrize("order", ["heads first", "padded", "one page", "one head"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_attention_of_pools_of_other_strides(built_lib, order, D):
    """Pools [heads, pages, ...], pages with a gap behind them, a single page, a single head: what the tensor map is made of."""
    from mserve_b200 import ops
    H, page, lens = 3, 32, [300, 77]
    if order == "one page":
        lens = [20]
    if order == "one head":
        H = 1
    src, table, g = _filled(len(lens), H, D, page, E4M3, lens, seed=D, spare=0 if order == "one page" else 3)
    if order == "one page":
        src = ops.Kv8Pages(*(t[int(table[0, 0])].unsqueeze(0).contiguous() for t in src))
        table = torch.zeros(1, 1, dtype=torch.int32)
    P = src.k.shape[0]

    def pool(t):
        if order == "heads first":
            return t.view(torch.uint8).transpose(0, 1).contiguous().transpose(0, 1).view(E4M3)
        gap = torch.full((P, H * page * D + 48), 0x7f, dtype=torch.uint8, device="cuda")       # NaN codes in the gap
        v = gap[:, :H * page * D].view(P, H, page, D)
        v.copy_(t.view(torch.uint8))
        return v.view(E4M3)

    pages = ops.Kv8Pages(pool(src.k), pool(src.v), src.exps, src.bounds)
    q = torch.randn(len(lens), 2 * H, 2, D, generator=g).to(BF16).cuda()
    want = ops.kv8_attention(q, src, table.cuda(), lens=_i32(lens))
    assert torch.equal(ops.kv8_attention(q, pages, table.cuda(), lens=_i32(lens)), want)
    ops.check_status(torch.device("cuda"))
