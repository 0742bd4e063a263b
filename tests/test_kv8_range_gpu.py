"""The 8-bit cache's attention where the softmax weights span many powers of two: pages of very different V scales,
scores far below the largest.

Scores here are exact: q is one at element 0 and zero elsewhere, K's element 0 a multiple of 1/8 that is a code, scale = ln 2,
so the weights are 2 to multiples of 1/8.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def _case(D, page, v, k0, cache, rows, dtype):
    """One sequence of v.shape[0] tokens, V = v, K = k0 at element 0; output [rows, D] in 64 bits and the exact one."""
    from mserve_b200 import ops
    n = v.shape[0]
    width = -(-n // page)
    pages = ops.kv8_pages(width, 1, D, page_size=page, dtype=cache)
    table = torch.arange(width, dtype=torch.int32, device="cuda").view(1, -1)
    k = torch.zeros(n, D)
    k[:, 0] = k0
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    ops.kv8_append(pages, table, k.view(1, 1, n, D).cuda(), v.float().view(1, 1, n, D).cuda(), tok0=torch.zeros_like(lens))
    exps = pages.exps.cpu().double()
    back = pages.v.cpu().double() * torch.pow(2.0, exps[:, :, 1])[..., None, None]
    assert torch.equal(back.view(-1, D)[:n], v.double()), "the case's values are codes"
    keys = pages.k.cpu().double() * torch.pow(2.0, exps[:, :, 0])[..., None, None]
    assert torch.equal(keys.view(-1, D)[:n, 0], k0.double())
    q = torch.zeros(1, rows, 1, D, dtype=dtype)
    q[..., 0] = 1
    out = ops.kv8_attention(q.cuda(), pages, table, lens=lens, scale=math.log(2)).cpu().double().view(rows, D)
    ops.check_status(torch.device("cuda"))
    w = torch.pow(2.0, k0.double() - k0.double().max())
    return out, (w[:, None] * v.double()).sum(dim=0) / w.sum(), exps[:, 0, 1].repeat_interleave(page)[:n], w


def _half_step(x, dtype):
    """Half the distance of neighbours of the type at x (normal values)."""
    bits = 8 if dtype == BF16 else 11
    return torch.pow(2.0, torch.frexp(x.abs())[1].double() - 1 - bits)


def _check(out, want, v, ev, w, dtype):
    # per weight: exponent arithmetic (|t| <= 64: 2^-18 in t, so 2^-18 of the weight), ex2 2^-22; the fp16 form 2^-11,
    # two terms 2^-21, and 2^-32 of the largest weight with its scale; sums of at most 40 terms: 40 * 2^-22 each way
    rel = 2.0 ** -17 + 80 * 2.0 ** -22 + 2.0 ** (-11 if dtype == BF16 else -21)
    scaled = w * torch.pow(2.0, ev)
    floor = 2.0 ** -32 * scaled.max() * (v.double().abs() / torch.pow(2.0, ev)[:, None]).sum(dim=0) / w.sum()
    tol = rel * (w[:, None] * v.double().abs()).sum(dim=0) / w.sum() + floor + _half_step(want, dtype)
    off = (out - want).abs()
    assert (off <= tol).all(), (float((off / tol).max()), float(((out - want) / want).abs().max()))
    return float((floor / want.abs()).max())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("cache", [torch.float8_e4m3fn, torch.float8_e5m2])
@pytest.mark.parametrize("D,rows", [(64, 1), (64, 12), (128, 3), (128, 16), (256, 5)])
@pytest.mark.parametrize("up", [0, 6, 12, 18, 20])
def test_one_outlier_channel(built_lib, dtype, cache, D, rows, up):
    """A page whose V has one channel 2^up larger: the other channels still are the mean over all pages.  Two tiles of one
    warp (tokens 0 to 15 and 128 to 143 of a CTA that takes all), the outlier in the first or in the second."""
    page, n = 16, 160
    g = torch.Generator().manual_seed(up)
    for where in (0, 128):
        v = (8 + torch.randint(0, 8, (n, D), generator=g)).double() / 8           # 1 to 1.875: codes in both types but for 1/8 steps
        if cache == torch.float8_e5m2:
            v = torch.floor(v * 4) / 4
        v[where:where + 16] = 0
        v[where:where + 16, 5] = 2.0 ** up if dtype == BF16 else 2.0 ** min(up, 12)
        k0 = torch.randint(0, 8, (n,), generator=g).double() / 4
        out, want, ev, w = _case(D, page, v, k0, cache, rows, dtype)
        _check(out, want.expand(rows, D), v, ev, w, dtype)


@pytest.mark.parametrize("lead,dtype", [(4, BF16), (4, F16), (11, F16), (14, BF16), (14, F16), (16, BF16), (16, F16), (20, BF16)])
def test_leading_token_of_zeros(built_lib, lead, dtype):
    """One token whose weight is 2^lead times the others' and whose V is zero: what is left is the others' small part."""
    D, n = 128, 16
    g = torch.Generator().manual_seed(lead)
    v = (8 + torch.randint(0, 8, (n, D), generator=g)).double() / 8
    v[3] = 0
    k0 = torch.randint(0, 16, (n,), generator=g).double() / 8
    k0[3] = lead
    out, want, ev, w = _case(D, 16, v, k0, torch.float8_e4m3fn, 2, dtype)
    assert dtype == BF16 or float(want.min()) >= 2.0 ** -14          # normal fp16 outputs
    share = _check(out, want.expand(2, D), v, ev, w, dtype)
    assert share < 2.0 ** -9
