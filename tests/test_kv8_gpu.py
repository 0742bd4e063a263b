"""The 8-bit paged cache's kernels (mskv_kv8_*) against the 64-bit oracle.

Appends are compared bit for bit (every code has one rounding).  Scores and attention are held to
bounds derived from the arithmetic (oracle.kv8_oracle), plus half a step of the output's type.
"""
import math

import pytest
import torch

from oracle import kv8_oracle as k8

pytestmark = pytest.mark.gpu

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2


def _host(pages):
    return {"k": pages.k.cpu().double(), "v": pages.v.cpu().double(), "exps": pages.exps.cpu().long(),
            "bounds": pages.bounds.cpu().double()}


def _same(pages, want):
    got = _host(pages)
    for name in ("exps", "k", "v", "bounds"):
        assert torch.equal(torch.nan_to_num(got[name].double(), nan=1e9), torch.nan_to_num(want[name].double(), nan=1e9)), name


def _table(B, width, spare, g):
    return torch.randperm(B * width + spare, generator=g)[:B * width].to(torch.int32).view(B, width)


def _filled(B, H, D, page, dtype, lens, seed, spare=3, size=1.0):
    """Pages holding random tokens for every sequence, through the append itself; (pages, table, generator)."""
    from mserve_b200 import ops
    g = torch.Generator().manual_seed(seed)
    width = max(lens) // page + 2
    table = _table(B, width, spare, g)
    pages = ops.kv8_pages(B * width + spare, H, D, page_size=page, dtype=dtype)
    n = max(max(lens), 1)
    scale = torch.exp2(torch.randint(-2, 3, (1, H, 1, D), generator=g).float()) * size
    k = torch.randn(B, H, n, D, generator=g) * scale
    v = torch.randn(B, H, n, D, generator=g) * torch.exp2(torch.randint(-4, 5, (1, 1, n, 1), generator=g).float())
    ops.kv8_append(pages, table.cuda(), k.cuda(), v.cuda(), tok0=torch.zeros(B, dtype=torch.int32, device="cuda"),
                   counts=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    ops.check_status(torch.device("cuda"))
    return pages, table, g


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ---- append ------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("new", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 16), (128, 48), (256, 32), (128, 128), (64, 64), (256, 128)])
def test_append_matches_definition(built_lib, dtype, new, D, page):
    """Several appends in a row: from nothing, into pages half full (exponents grow and shrink), ragged, none."""
    from mserve_b200 import ops
    B, H = 4, 3
    g = torch.Generator().manual_seed(D * 1000 + page)
    width = 6
    table = _table(B, width, 2, g)
    pages = ops.kv8_pages(B * width + 2, H, D, page_size=page, dtype=dtype)
    want = _host(pages)
    tok0 = torch.zeros(B, dtype=torch.int32)
    for step, counts in enumerate([[1, page, 2 * page + 5, 0], [1, 1, 1, 1], [page - 2, 3, 0, page + 1], [1, 0, 7, 1]]):
        n = max(counts)
        mag = 10.0 ** float(torch.randint(-6, 4, (1,), generator=g))
        k = (torch.randn(B, H, n, D, generator=g) * mag).to(new)
        v = (torch.randn(B, H, n, D, generator=g) / mag).to(new)
        cnt = torch.tensor(counts, dtype=torch.int32)
        for _ in range(2):      # repeating a call changes nothing
            ops.kv8_append(pages, table.cuda(), k.cuda(), v.cuda(), tok0=tok0.cuda(), counts=cnt.cuda())
            if _ == 0:
                want = k8.append(want, table, k.double(), v.double(), tok0, cnt, dtype)
            _same(pages, want)
        tok0 += cnt
    ops.check_status(torch.device("cuda"))


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
def test_append_special_values(built_lib, dtype):
    """Zeros, subnormals, values on a code's border, infinities, NaN, values beyond the exponents' range."""
    from mserve_b200 import ops
    D, page, H = 64, 16, 1
    bits, least, largest = k8.F8[dtype]
    rows = torch.zeros(8 * page, D)
    rows[page] = torch.linspace(-largest, largest, D)                       # exactly the largest code
    rows[2 * page] = torch.linspace(-largest, largest, D) * (1 + 2.0 ** -20)  # just above it
    rows[3 * page, :4] = torch.tensor([math.inf, -math.inf, math.nan, 3.0])
    rows[4 * page, :3] = torch.tensor([1e38, -1e38, 1.0])                   # saturates at the largest exponent
    rows[5 * page, :3] = torch.tensor([1e-40, -1e-30, 1e-25])               # below the smallest
    steps = torch.arange(D) * 2.0 ** (least - bits - 1)                     # subnormal codes and their halves
    rows[6 * page] = steps
    rows[6 * page + 1, 0] = largest
    rows[7 * page, 0] = math.nan
    table = torch.arange(8, dtype=torch.int32).view(1, 8)
    pages = ops.kv8_pages(8, H, D, page_size=page, dtype=dtype)
    x = rows.view(1, 1, 8 * page, D)
    ops.kv8_append(pages, table.cuda(), x.cuda(), x.cuda(), tok0=_i32([0]))
    want = k8.append(_host(ops.kv8_pages(8, H, D, page_size=page, dtype=dtype)), table, x.double(), x.double(), [0], [8 * page], dtype)
    _same(pages, want)
    assert int(pages.exps[0, 0, 0]) == k8.EXP_MIN and int(pages.exps[1, 0, 0]) == 0 and int(pages.exps[2, 0, 0]) == 1


@pytest.mark.parametrize("new", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("page", [16, 64])
def test_append_infinities_in_one_half(built_lib, new, page):
    """Infinities and NaN in K or in V alone, in pages of new rows only and in pages that also hold old ones."""
    from mserve_b200 import ops
    H, D = 2, 128
    g = torch.Generator().manual_seed(77)
    for where in ("k", "v"):
        table = torch.arange(4, dtype=torch.int32).view(1, 4)
        pages = ops.kv8_pages(4, H, D, page_size=page)
        want = _host(pages)
        tok0 = 0
        for n in (2 * page - 5, 9, page):
            rows = {name: torch.randn(1, H, n, D, generator=g) for name in ("k", "v")}
            rows[where][0, 0, n // 2, 3] = math.inf
            rows[where][0, 1, n - 1, 5] = -math.inf
            rows[where][0, 1, 0, 7] = math.nan
            rows = {name: t.to(new) for name, t in rows.items()}
            ops.kv8_append(pages, table.cuda(), rows["k"].cuda(), rows["v"].cuda(), tok0=_i32([tok0]))
            want = k8.append(want, table, rows["k"].double(), rows["v"].double(), [tok0], [n], E4M3)
            _same(pages, want)
            tok0 += n
    ops.check_status(torch.device("cuda"))


def test_append_strides_and_rows_behind(built_lib):
    """Token-major, unaligned and broadcast rows; pools inside one allocation; rows behind the end keep their bytes."""
    from mserve_b200 import ops
    B, H, D, page, n = 3, 2, 128, 32, 21
    g = torch.Generator().manual_seed(5)
    both = torch.randint(0, 120, (12, 2, H, page, D), dtype=torch.uint8, generator=g).cuda()
    pool = both.view(E4M3)
    pages = ops.Kv8Pages(pool[:, 0], pool[:, 1], torch.zeros(12, H, 2, dtype=torch.int8, device="cuda"),
                         torch.zeros(12, H, 2, D, dtype=torch.uint8, device="cuda").view(E4M3))
    table = _table(B, 3, 3, g)
    tok0 = torch.tensor([0, 5, 30], dtype=torch.int32)
    fused = torch.randn(B, n, 3 * H * D + 1, generator=g).to(torch.bfloat16).cuda()
    k = fused[:, :, 1:1 + H * D].view(B, n, H, D).transpose(1, 2)           # 2-byte aligned
    v = fused[:, :1, 1 + H * D:1 + 2 * H * D].view(B, 1, H, D).transpose(1, 2).expand(B, H, n, D)
    want = k8.append(_host(pages), table, k.cpu().double(), v.cpu().double(), tok0, [n] * B, E4M3)
    ops.kv8_append(pages, table.cuda(), k, v, tok0=tok0.cuda())
    _same(pages, want)
    ops.check_status(torch.device("cuda"))


def test_append_bad_destinations(built_lib):
    """Unmapped and foreign pages, negative positions and tokens past the table: skipped, reported, nothing else touched."""
    from mserve_b200 import ops
    H, D, page = 2, 64, 16
    pages = ops.kv8_pages(4, H, D, page_size=page)
    dev = torch.device("cuda")
    x = torch.ones(1, H, 20, D, device="cuda")
    for table, tok0, counts, word, kept in [([[0, -1]], 0, 20, "not mapped", 16), ([[0, 4]], 0, 20, "not mapped", 16),
                                            ([[0, 1]], -3, 20, "destination", 0), ([[0, 1]], 30, 20, "destination", 2),
                                            ([[0, 1]], 2 ** 31 - 20, 20, "destination", 0)]:
        for t in pages[:3]:
            t.view(torch.uint8).zero_()
        ops.kv8_append(pages, _i32(table), x, x, tok0=_i32([tok0]), counts=_i32([counts]))
        with pytest.raises(RuntimeError, match=word):
            ops.check_status(dev)
        assert int((pages.k.float() != 0).sum()) == kept * H * D, (table, tok0)
    ops.kv8_append(pages, _i32([[0, 1]]), x, x, tok0=_i32([0]), counts=_i32([-5]))     # a negative count is none
    ops.check_status(dev)


# ---- block scores ------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,qt", [(E4M3, torch.bfloat16), (E4M3, torch.float16), (E5M2, torch.bfloat16)])
@pytest.mark.parametrize("H,G,D,page,lens", [(2, 7, 128, 16, [0, 1, 16, 17, 1000]), (1, 1, 64, 32, [777]),
                                             (3, 5, 256, 16, [2100, 5]), (2, 16, 128, 128, [130, 129, 128])])
def test_block_scores(built_lib, dtype, qt, H, G, D, page, lens):
    from mserve_b200 import ops
    B = len(lens)
    pages, table, g = _filled(B, H, D, page, dtype, lens, seed=D + page)
    q = (torch.randn(B, H * G, D, generator=g) * torch.exp2(torch.randint(-9, 6, (1, 1, D), generator=g).float())).to(qt)
    nb = table.shape[1]
    out = torch.full((B, H, nb + 3), 7.0, device="cuda")
    ops.kv8_block_score(q.cuda(), pages, table.cuda(), lens=_i32(lens), max_blocks=nb, out=out)
    ops.check_status(torch.device("cuda"))
    want, mag = k8.block_scores(q.double(), _host(pages), table, lens)
    got = out.cpu().double()
    held = torch.isfinite(want)
    assert (got[:, :, nb:] == 7).all() and (got[:, :, :nb][~held] == 7).all()
    # 2D products in fp32: 2D/16 + 4 roundings of at most 2^-22 of the magnitudes; the weights keep 23 bits of
    # the largest: 2^-23 of (largest weight * sum of code magnitudes) <= 2^-23 * 2D * largest weight * largest code
    host = _host(pages)
    code = torch.stack([torch.stack([host["bounds"][table[b].long(), h].abs().sum(dim=(1, 2))
                                     * torch.pow(2.0, host["exps"][table[b].long(), h, 0].double()) for h in range(H)])
                        for b in range(B)])                                  # [B, H, nb]
    w = q.double().abs().view(B, H, G, D).sum(dim=2).amax(dim=-1)[..., None]
    tol = mag * (2 * D / 16 + 4) * 2.0 ** -22 + code * w * 2.0 ** -23 + G * mag * 2.0 ** -24
    off = (got[:, :, :nb] - want).abs()
    assert (off[held] <= tol[held]).all(), float((off / tol)[held].max())
    # no token of a block has a larger GQA-summed q.k
    for b in range(B):
        for h in range(H):
            for j in range(-(-lens[b] // page)):
                rows = host["k"][int(table[b, j]), h, :min(page, lens[b] - j * page)] * 2.0 ** int(host["exps"][int(table[b, j]), h, 0])
                s = (q[b, h * G:(h + 1) * G].double() @ rows.T).sum(dim=0).max()
                assert s <= got[b, h, j] + tol[b, h, j]


def test_block_scores_bad_page_and_bound(built_lib):
    from mserve_b200 import ops
    pages, table, g = _filled(1, 2, 64, 16, E4M3, [100], seed=1)
    q = torch.randn(1, 4, 64, generator=g).to(torch.bfloat16).cuda()
    t = table.clone()
    t[0, 2], t[0, 5] = -1, pages.k.shape[0]
    out = torch.zeros(1, 2, 4, device="cuda")
    ops.kv8_block_score(q, pages, t.cuda(), lens=_i32([100]), max_blocks=4, out=out)     # lens beyond max_blocks: clamped
    with pytest.raises(RuntimeError, match="not mapped"):
        ops.check_status(torch.device("cuda"))
    assert torch.isinf(out[0, :, 2]).all() and torch.isfinite(out[0, :, [0, 1, 3]]).all()
    pages.bounds[int(table[0, 1]), 0, 0, 3] = float("nan")
    ops.kv8_block_score(q, pages, table.cuda(), lens=_i32([64]), max_blocks=4, out=out)
    assert torch.isnan(out[0, 0, 1]) and torch.isfinite(out[0, 1]).all() and torch.isfinite(out[0, 0, [0, 2, 3]]).all()
    ops.check_status(torch.device("cuda"))


# ---- attention ---------------------------------------------------------------------------------
def _close(got, want, bound):
    g = got.cpu().double()
    tol = bound * 1.0 + want.abs() * torch.finfo(got.dtype).eps / 2 + (2.0 ** -25 if got.dtype == torch.float16 else 0)
    off = (g - want).abs()
    assert torch.isfinite(g).all()
    assert (off <= tol).all(), (float((off / tol.clamp(min=1e-300)).max()), float(off.max()))


def _bits(qt):
    return 11 if qt == torch.bfloat16 else 21


LENS = [[0, 1, 15, 16], [17, 255, 256, 257], [1000, 3, 64], [5000]]


@pytest.mark.parametrize("dtype,qt", [(E4M3, torch.bfloat16), (E4M3, torch.float16), (E5M2, torch.bfloat16), (E5M2, torch.float16)])
@pytest.mark.parametrize("H,G,D,page,Q", [(2, 7, 128, 16, 1), (1, 1, 64, 32, 1), (2, 5, 256, 16, 1), (1, 12, 128, 64, 1),
                                          (2, 4, 64, 16, 4), (1, 7, 128, 48, 16), (1, 3, 256, 128, 5), (3, 16, 64, 16, 2)])
@pytest.mark.parametrize("lens", LENS)
def test_attention(built_lib, dtype, qt, H, G, D, page, Q, lens):
    from mserve_b200 import ops
    B = len(lens)
    pages, table, g = _filled(B, H, D, page, dtype, lens, seed=sum(lens) + D)
    q = (torch.randn(B, H * G, Q, D, generator=g) * 0.5).to(qt)
    out = ops.kv8_attention(q.cuda(), pages, table.cuda(), lens=_i32(lens), max_tokens=max(lens))
    ops.check_status(torch.device("cuda"))
    assert out.shape == q.shape and out.dtype == qt
    want, bound = k8.attention(q.double(), _host(pages), table, lens, weight_bits=_bits(qt))
    _close(out, want, bound)
    for b, n in enumerate(lens):
        for i in range(Q):
            if n - Q + 1 + i <= 0:
                assert (out[b, :, i] == 0).all()
    # a looser bound on the lengths may split the work differently, never change what is computed
    _close(ops.kv8_attention(q.cuda(), pages, table.cuda(), lens=_i32(lens)), want, bound)


@pytest.mark.parametrize("dtype,qt", [(E4M3, torch.bfloat16), (E5M2, torch.float16)])
@pytest.mark.parametrize("H,G,D,page,Q,lens,S", [(2, 7, 128, 16, 1, [0, 1, 500, 2000], 9), (4, 5, 128, 16, 1, [3000] * 3, 150),
                                                 (2, 4, 64, 64, 3, [700, 65], 5), (1, 12, 256, 32, 1, [1500, 40], 20)])
def test_attention_over_blocks(built_lib, dtype, qt, H, G, D, page, Q, lens, S):
    """Lists in any order, with repeats, of any count; entries behind the count are not read."""
    from mserve_b200 import ops
    B = len(lens)
    pages, table, g = _filled(B, H, D, page, dtype, lens, seed=sum(lens) + S)
    blocks = torch.full((B, H, S), 2 ** 30, dtype=torch.int32)
    counts = torch.zeros(B, H, dtype=torch.int32)
    for b in range(B):
        held = -(-lens[b] // page)
        for h in range(H):
            n = int(torch.randint(0, S + 1, (1,), generator=g)) if held and (b, h) != (B - 1, 0) else (S if held else 0)
            counts[b, h] = n
            if n:
                blocks[b, h, :n] = torch.randint(0, held, (n,), generator=g)
    q = torch.randn(B, H * G, Q, D, generator=g).to(qt)
    out = ops.kv8_attention(q.cuda(), pages, table.cuda(), lens=_i32(lens), blocks=blocks.cuda(), counts=counts.cuda())
    ops.check_status(torch.device("cuda"))
    want, bound = k8.attention(q.double(), _host(pages), table, lens, blocks=blocks, counts=counts, weight_bits=_bits(qt))
    _close(out, want, bound)


def test_attention_all_blocks_equal_whole(built_lib):
    from mserve_b200 import ops
    pages, table, g = _filled(2, 2, 128, 16, E4M3, [900, 333], seed=3)
    q = torch.randn(2, 14, 1, 128, generator=g).to(torch.bfloat16).cuda()
    blocks = torch.arange(57, dtype=torch.int32, device="cuda").view(1, 1, -1).expand(2, 2, -1)     # broadcast lists
    whole = ops.kv8_attention(q, pages, table.cuda(), lens=_i32([900, 333]))
    listed = ops.kv8_attention(q, pages, table.cuda(), lens=_i32([900, 333]), blocks=blocks)        # pages behind 333: no tokens
    ops.check_status(torch.device("cuda"))
    assert (whole.float() - listed.float()).abs().max() <= 2 ** -7 * whole.float().abs().max()
    none = ops.kv8_attention(q, pages, table.cuda(), lens=_i32([900, 333]), blocks=blocks[:, :, :0])
    assert (none == 0).all()


def test_attention_strides_scale_and_out(built_lib):
    """Transposed and unaligned queries, a given out, negative and zero scales, cache halves of one allocation."""
    from mserve_b200 import ops
    lens = [321, 40]
    src, table, g = _filled(2, 2, 128, 16, E4M3, lens, seed=11)
    both = torch.stack([src.k.view(torch.uint8), src.v.view(torch.uint8)], dim=1).view(E4M3)
    pages = ops.Kv8Pages(both[:, 0], both[:, 1], src.exps, None)
    buf = torch.randn(2, 3, 6 * 128 + 1, generator=g).to(torch.bfloat16)
    for off in (0, 1):
        q = buf[:, :, off:off + 6 * 128].view(2, 3, 6, 128).transpose(1, 2)
        hold = torch.full((2, 3, 6 * 128 + 1), 5.0, dtype=torch.bfloat16, device="cuda")
        out = hold[:, :, off:off + 6 * 128].view(2, 3, 6, 128).transpose(1, 2)
        for scale in (0.1, -0.2, 0.0):
            dq = buf.cuda()[:, :, off:off + 6 * 128].view(2, 3, 6, 128).transpose(1, 2)
            r = ops.kv8_attention(dq, pages, table.cuda(), lens=_i32(lens), scale=scale, out=out)
            assert r.data_ptr() == out.data_ptr()
            want, bound = k8.attention(q.double(), _host(src), table, lens, scale=scale)
            _close(out, want, bound)
        edge = hold[:, :, 6 * 128 if off == 0 else 0]
        assert (edge == 5).all()


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
def test_attention_masked_places(built_lib, dtype):
    """NaN codes behind the sequences and in unlisted pages change nothing; a NaN V of a token reaches exactly
    the positions that see it; a NaN K makes their rows NaN."""
    from mserve_b200 import ops
    B, H, G, D, page, Q = 2, 2, 3, 64, 16, 4
    lens = [70, 18]
    pages, table, g = _filled(B, H, D, page, dtype, lens, seed=8)
    q = torch.randn(B, H * G, Q, D, generator=g).to(torch.bfloat16).cuda()
    clean = ops.kv8_attention(q, pages, table.cuda(), lens=_i32(lens))
    nan = 0x7f
    used = torch.zeros(pages.k.shape[0], page, dtype=torch.bool)
    for b in range(B):
        for t in range(lens[b]):
            used[int(table[b, t // page]), t % page] = True
    for pool in (pages.k, pages.v):
        pool.view(torch.uint8)[(~used).cuda()[:, None].expand(-1, H, -1)] = nan
    assert torch.equal(ops.kv8_attention(q, pages, table.cuda(), lens=_i32(lens)), clean)
    # token 68 of sequence 0 (seen by positions 2 and 3: tokens < 70 - 4 + 1 + i), dim 5 of head 1
    pid = int(table[0, 68 // page])
    pages.v.view(torch.uint8)[pid, 1, 68 % page, 5] = nan
    out = ops.kv8_attention(q, pages, table.cuda(), lens=_i32(lens))
    bad = torch.isnan(out)
    want = torch.zeros_like(bad)
    want[0, G:2 * G, 2:, 5] = True
    assert torch.equal(bad, want)
    assert torch.equal(out[~bad], clean[~bad])
    pages.v.view(torch.uint8)[pid, 1, 68 % page, 5] = 0
    pages.k.view(torch.uint8)[pid, 1, 68 % page, 5] = nan
    out = ops.kv8_attention(q, pages, table.cuda(), lens=_i32(lens))
    want = torch.zeros_like(bad)
    want[0, G:2 * G, 2:] = True
    assert torch.equal(torch.isnan(out), want)
    # first token: seen by all
    pages.k.view(torch.uint8)[pid, 1, 68 % page, 5] = 0
    pages.v.view(torch.uint8)[int(table[1, 0]), 0, 0, 9] = nan
    out = ops.kv8_attention(q, pages, table.cuda(), lens=_i32(lens))
    want = torch.zeros_like(bad)
    want[1, :G, :, 9] = True
    assert torch.equal(torch.isnan(out), want)
    ops.check_status(torch.device("cuda"))


def test_attention_wide_exponents(built_lib):
    """Pages whose scales differ by up to 2^60 and all-zero pages: no term of weight is lost."""
    from mserve_b200 import ops
    H, D, page, n = 1, 64, 16, 16 * 6
    g = torch.Generator().manual_seed(4)
    pages = ops.kv8_pages(6, H, D, page_size=page)
    table = torch.arange(6, dtype=torch.int32).view(1, 6)
    k, v = torch.randn(1, H, n, D, generator=g), torch.randn(1, H, n, D, generator=g)
    for p, mag in enumerate([1.0, 0.0, 2.0 ** 20, 2.0 ** -40, 1.0, 2.0 ** -50]):
        v[:, :, p * page:(p + 1) * page] *= mag
    k[:, :, 5 * page:] *= 20
    ops.kv8_append(pages, table.cuda(), k.cuda(), v.cuda(), tok0=_i32([0]))
    q = torch.randn(1, 4, 1, D, generator=g).to(torch.bfloat16)
    for size in (1.0, 30.0):
        qq = (q.float() * size).to(torch.bfloat16)
        out = ops.kv8_attention(qq.cuda(), pages, table.cuda(), lens=_i32([n]))
        want, bound = k8.attention(qq.double(), _host(pages), table, [n])
        _close(out, want, bound)


def test_attention_bad_entries(built_lib):
    from mserve_b200 import ops
    pages, table, g = _filled(1, 1, 64, 16, E4M3, [160], seed=2)
    dev = torch.device("cuda")
    q = torch.randn(1, 2, 1, 64, generator=g).to(torch.bfloat16).cuda()
    blocks = torch.tensor([[[0, -1, 3, 11, 12, 2 ** 31 - 1]]], dtype=torch.int32)     # table width 12
    out = ops.kv8_attention(q, pages, table.cuda(), lens=_i32([160]), blocks=blocks.cuda())
    with pytest.raises(RuntimeError, match="out of range"):
        ops.check_status(dev)
    good = ops.kv8_attention(q, pages, table.cuda(), lens=_i32([160]), blocks=_i32([[[0, 3]]]))
    assert torch.equal(out, good)
    t = table.clone()
    t[0, 1], t[0, 2] = -7, pages.k.shape[0]
    out = ops.kv8_attention(q, pages, t.cuda(), lens=_i32([160]))
    with pytest.raises(RuntimeError, match="not mapped"):
        ops.check_status(dev)
    good = ops.kv8_attention(q, pages, table.cuda(), lens=_i32([160]), blocks=_i32([[[0, 3, 4, 5, 6, 7, 8, 9]]]))
    assert (out.float() - good.float()).abs().max() <= 2 ** -7 * good.float().abs().max()
    # lengths beyond the bound and below zero are clamped
    a = ops.kv8_attention(q, pages, table.cuda(), lens=_i32([10 ** 9]), max_tokens=100)
    b = ops.kv8_attention(q, pages, table.cuda(), lens=_i32([100]), max_tokens=100)
    assert torch.equal(a, b)
    assert (ops.kv8_attention(q, pages, table.cuda(), lens=_i32([-4])) == 0).all()
    ops.check_status(dev)


def test_many_ragged_sequences(built_lib):
    """More sequences than CTAs, most of them short or empty: every segment is written once."""
    from mserve_b200 import ops
    g = torch.Generator().manual_seed(9)
    lens = torch.randint(0, 60, (400,), generator=g).tolist()
    lens[7], lens[201], lens[399] = 4000, 300, 0
    pages, table, g = _filled(400, 2, 64, 16, E4M3, lens, seed=12)
    q = torch.randn(400, 6, 1, 64, generator=g).to(torch.bfloat16)
    out = torch.full(q.shape, float("nan"), dtype=q.dtype, device="cuda")
    ops.kv8_attention(q.cuda(), pages, table.cuda(), lens=_i32(lens), out=out)
    want, bound = k8.attention(q.double(), _host(pages), table, lens)
    _close(out, want, bound)


@pytest.mark.parametrize("B,H,G,D,Q,most,qt", [(80, 4, 7, 128, 1, 700, torch.bfloat16), (60, 4, 7, 128, 5, 900, torch.float16),
                                               (40, 3, 5, 256, 5, 700, torch.bfloat16), (30, 4, 12, 64, 5, 600, torch.float16)])
def test_several_waves_of_segments(built_lib, B, H, G, D, Q, most, qt):
    """More segments than CTAs at once, short ones: a CTA takes each from its first to its last token."""
    from mserve_b200 import ops
    g = torch.Generator().manual_seed(D + Q)
    lens = torch.randint(0, most + 1, (B,), generator=g).tolist()
    lens[0], lens[1], lens[-1] = most, 0, 1
    pages, table, g = _filled(B, H, D, 32, E4M3, lens, seed=D)
    q = (torch.randn(B, H * G, Q, D, generator=g) * 0.5).to(qt)
    out = torch.full(q.shape, float("nan"), dtype=qt, device="cuda")
    ops.kv8_attention(q.cuda(), pages, table.cuda(), lens=_i32(lens), max_tokens=most, out=out)
    ops.check_status(torch.device("cuda"))
    want, bound = k8.attention(q.double(), _host(pages), table, lens, weight_bits=_bits(qt))
    _close(out, want, bound)


def test_large_offsets(built_lib):
    """Pools past 2^31 bytes, with the sequence's pages at both ends."""
    from mserve_b200 import ops
    H, D, page = 1, 128, 128
    P = 2 ** 31 // (page * D) + 40
    pages = ops.kv8_pages(P, H, D, page_size=page)
    table = torch.tensor([[P - 1, 0, P - 2, 131072, 131071]], dtype=torch.int32)
    g = torch.Generator().manual_seed(6)
    n = 5 * page - 7
    k, v = torch.randn(1, H, n, D, generator=g), torch.randn(1, H, n, D, generator=g)
    ops.kv8_append(pages, table.cuda(), k.cuda(), v.cuda(), tok0=_i32([0]))
    small = ops.Kv8Pages(*(t.view(torch.uint8)[table[0].long().cuda()].view(t.dtype).contiguous() for t in pages))
    order = torch.arange(5, dtype=torch.int32).view(1, 5)
    want = k8.append(_host(ops.kv8_pages(5, H, D, page_size=page)), order, k.double(), v.double(), [0], [n], E4M3)
    _same(small, want)
    q = torch.randn(1, 2, 1, D, generator=g).to(torch.bfloat16)
    out = ops.kv8_attention(q.cuda(), pages, table.cuda(), lens=_i32([n]))
    ref, bound = k8.attention(q.double(), want, order, [n])
    _close(out, ref, bound)
    s = torch.zeros(1, 1, 5, device="cuda")
    ops.kv8_block_score(q.cuda(), pages, table.cuda(), lens=_i32([n]), max_blocks=5, out=s)
    s2 = torch.zeros_like(s)
    ops.kv8_block_score(q.cuda(), small, order.cuda(), lens=_i32([n]), max_blocks=5, out=s2)
    assert torch.equal(s, s2)
    ops.check_status(torch.device("cuda"))


@pytest.mark.parametrize("tokens", [2000, 9000])        # a cluster for each segment; the line and its merge
def test_streams_and_graphs(built_lib, tokens):
    """Calls on a side stream; two streams at once; two graphs of the same call on different inputs, replayed at the
    same time; a graph replayed while the cache grows."""
    from mserve_b200 import ops
    lens = [700, 1300]
    pages, table, g = _filled(2, 2, 128, 16, E4M3, [tokens, tokens], seed=21)
    table = table.cuda()
    qs = [torch.randn(2, 14, 1, 128, generator=g).to(torch.bfloat16).cuda() for _ in range(2)]
    n = _i32(lens)
    want = [ops.kv8_attention(q, pages, table, lens=n, max_tokens=tokens).clone() for q in qs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = ops.kv8_attention(qs[0], pages, table, lens=n, max_tokens=tokens, stream=side)
    side.synchronize()
    assert torch.equal(got, want[0])
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    both = [[ops.kv8_attention(q, pages, table, lens=n, max_tokens=tokens, stream=st) for q, st in zip(qs, streams)]
            for _ in range(10)]
    torch.cuda.synchronize()
    for pair in both:
        assert torch.equal(pair[0], want[0]) and torch.equal(pair[1], want[1])
    graphs, outs = [], []
    for q in qs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(ops.kv8_attention(q, pages, table, lens=n, max_tokens=tokens))
        graphs.append(gr)
    torch.cuda.synchronize()
    for _ in range(20):
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)
    n.copy_(_i32([tokens - 1, 5]))
    graphs[0].replay()
    assert torch.equal(outs[0], ops.kv8_attention(qs[0], pages, table, lens=n, max_tokens=tokens))
    torch.cuda.synchronize()
    ops.check_status(torch.device("cuda"))
    del graphs


def test_captured_across_streams(built_lib):
    """A graph whose streams fork and join between the calls: append on one, scores and attention on another."""
    from mserve_b200 import ops
    B, H, D, page = 2, 2, 128, 16
    pages, table, g = _filled(B, H, D, page, E4M3, [500, 90], seed=51)
    tab, tok0, n = table.cuda(), _i32([500, 90]), _i32([501, 91])
    x = torch.randn(2, B, H, 1, D, generator=g).to(torch.bfloat16).cuda()
    q = torch.randn(B, 14, 1, D, generator=g).to(torch.bfloat16).cuda()
    scores = torch.zeros(B, H, tab.shape[1], device="cuda")
    out = torch.zeros_like(q)
    side = torch.cuda.Stream()

    def work():
        main = torch.cuda.current_stream()
        ops.kv8_append(pages, tab, x[0], x[1], tok0=tok0)
        side.wait_stream(main)
        ops.kv8_block_score(q, pages, tab, lens=n, max_blocks=tab.shape[1], out=scores, stream=side)
        ops.kv8_attention(q, pages, tab, lens=n, out=out, stream=side)
        main.wait_stream(side)
        return out + 1

    work()
    torch.cuda.synchronize()
    want, s = out.clone(), scores.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plus = work()
    for _ in range(5):
        out.zero_()
        scores.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(plus, want + 1) and torch.equal(scores, s)
    ops.check_status(torch.device("cuda"))
    del graph


@pytest.mark.parametrize("D,Q", [(64, 1), (128, 1), (128, 4)])
def test_bounds_far_above_the_lengths(built_lib, D, Q):
    """A page table for a quarter of a million tokens with a few hundred in it: the work is split by the lengths."""
    from mserve_b200 import ops
    lens = [600, 0, 33, 599, 1, 350, 16, 17]
    pages, table, g = _filled(8, 2, D, 16, E4M3, lens, seed=61)
    wide = torch.full((8, 16000), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    q = torch.randn(8, 14, Q, D, generator=g).to(torch.bfloat16)
    want, bound = k8.attention(q.double(), _host(pages), table, lens)
    _close(ops.kv8_attention(q.cuda(), pages, wide.cuda(), lens=_i32(lens)), want, bound)
    ops.check_status(torch.device("cuda"))


def test_attention_of_extreme_scores(built_lib):
    """Scores of either sign far beyond what exp holds: a row whose scores are all very small is still a mean."""
    from mserve_b200 import ops
    pages, table, g = _filled(1, 1, 64, 16, E4M3, [80], seed=71)
    host = _host(pages)
    for size in (1e15, 1e30):
        q = torch.zeros(1, 2, 1, 64)
        q[0, 0, 0, 3], q[0, 1, 0, 3] = size, -size
        q = q.to(torch.bfloat16)
        want, _ = k8.attention(q.double(), host, table, [80])
        got = ops.kv8_attention(q.cuda(), pages, table.cuda(), lens=_i32([80])).cpu().double()
        # one token's weight is 1 (its score leads by more than 2^20 times the rounding of any): half a step of the output
        assert ((got - want).abs() <= want.abs() * 2.0 ** -8).all()


def test_results_do_not_vary(built_lib):
    """The same call gives the same bits every time (no atomics in any sum)."""
    from mserve_b200 import ops
    lens = [3333, 900, 17]
    pages, table, g = _filled(3, 2, 128, 16, E4M3, lens, seed=31)
    q = torch.randn(3, 14, 1, 128, generator=g).to(torch.float16).cuda()
    first = ops.kv8_attention(q, pages, table.cuda(), lens=_i32(lens))
    for _ in range(20):
        assert torch.equal(ops.kv8_attention(q, pages, table.cuda(), lens=_i32(lens)), first)


def test_selection_run_together(built_lib):
    """Append -> block scores -> top-k with the last blocks -> attention over the list, as a decode step runs them."""
    from mserve_b200 import ops
    B, H, G, D, page = 3, 2, 7, 128, 16
    lens = [1500, 47, 800]
    pages, table, g = _filled(B, H, D, page, E4M3, lens, seed=41)
    tab = table.cuda()
    x = torch.randn(2, B, H, 1, D, generator=g).to(torch.bfloat16).cuda()
    ops.kv8_append(pages, tab, x[0], x[1], tok0=_i32(lens))
    lens = [n + 1 for n in lens]
    n = _i32(lens)
    held = (n + page - 1) // page
    q = torch.randn(B, H * G, 1, D, generator=g).to(torch.bfloat16)
    nb, K, R = tab.shape[1], 10, 2
    scores = torch.zeros(B, H, nb, device="cuda")
    ops.kv8_block_score(q.cuda(), pages, tab, lens=n, max_blocks=nb, out=scores)
    idx, counts = ops.topk(scores.view(B * H, nb), top_k=K, recent=R, len_=held.to(torch.int32), len_scalar=nb, sel_per_batch=H)
    idx, counts = idx.view(B, H, -1), counts.view(B, H)
    out = ops.kv8_attention(q.cuda(), pages, tab, lens=n, blocks=idx, counts=counts)
    ops.check_status(torch.device("cuda"))
    for b in range(B):
        nblk = -(-lens[b] // page)
        for h in range(H):
            sel = idx[b, h, :int(counts[b, h])].tolist()
            assert sel == sorted(sel) and len(sel) == min(K, max(nblk - R, 0)) + min(R, nblk)
            assert sel[-min(R, nblk):] == list(range(nblk - min(R, nblk), nblk))
            cand = scores[b, h, :max(nblk - R, 0)].cpu()
            assert set(sel[:len(sel) - min(R, nblk)]) == set(cand.topk(min(K, cand.numel())).indices.tolist())
    want, bound = k8.attention(q.double(), _host(pages), table, lens, blocks=idx.cpu(), counts=counts.cpu())
    _close(out, want, bound)
