"""Cases of the 8-bit paged KV cache: its append, its attention (whole and over selected blocks), its block scores.

The cache holds keys and values as 8-bit floats in pages of tokens, ``k``/``v`` [pages, KV heads, page, D], with one
power-of-two scale per (page, KV head): ``exps`` int8 [pages, KV heads, 2] (keys, values), value = code * 2^exp, and the
elementwise minimum and maximum of every page's key codes, ``bounds`` [pages, KV heads, 2, D].  A page table
[batch, pages of a sequence] maps logical pages to physical ones.

``own`` false: the operators in elementary torch operations.  ``own`` true: the package's kernels.
"""
import math

import torch

own = False

LOW, HIGH = -60, 60                                   # range of the exponents
LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}            # largest finite code
CACHE = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _case(name, op, batch, q_heads, kv_heads, tokens, *, head_dim=128, page=16, q_len=1, ragged=False, dtype="bf16",
          cache="e4m3", new=0, blocks=0, recent=0, token_major=False):
    named = {} if name is None else {"name": name}
    return {**named, "op": op, "batch": batch, "q_heads": q_heads, "kv_heads": kv_heads, "tokens": tokens,
            "head_dim": head_dim, "page": page, "q_len": q_len, "ragged": ragged, "dtype": dtype, "cache": cache,
            "new": new, "blocks": blocks, "recent": recent, "token_major": token_major}


def listed():
    return [
        # one decode step's token of 8 sequences, written into pages that already hold some (28/4 heads)
        _case("append token", "append", 8, 28, 4, 16384, new=1, ragged=True),
        # a conversation turn of up to 64 text tokens, rows as a fused projection leaves them (token-major, f16)
        _case("append turn", "append", 4, 56, 8, 4100, new=64, ragged=True, dtype="f16", page=32, token_major=True),
        # a long prompt going into the cache
        _case("append prompt", "append", 2, 40, 8, 0, new=16384),
        # the smallest decode: one sequence that has just begun
        _case("attend short", "attend", 1, 28, 4, 33),
        # decode of 8 sequences of 16384 tokens, 28/4 heads
        _case("attend 16k", "attend", 8, 28, 4, 16384),
        # decode of 16 sequences of 32768 tokens, 40/8 heads
        _case("attend 32k", "attend", 16, 40, 8, 32768),
        # four proposed tokens checked at once over ragged sequences; small heads, larger pages, the wide 8-bit type
        _case("attend verify ragged", "attend", 6, 32, 8, 9001, head_dim=64, page=32, q_len=4, ragged=True, dtype="f16",
              cache="e5m2"),
        # block scores of one decode step: 8 sequences of 16384 tokens, 28/4 heads
        _case("score 16k", "score", 8, 28, 4, 16384),
        # block scores of 16 sequences of up to 65536 tokens, 56/8 heads
        _case("score 64k ragged", "score", 16, 56, 8, 65536, ragged=True),
        # selected blocks of the 28/4 decode: 2048 tokens and the last 128
        _case("blocks 16k", "blocks", 8, 28, 4, 16384, blocks=128, recent=8),
        # selected blocks of the 40/8 decode: 4096 tokens and the last 256
        _case("blocks 32k", "blocks", 16, 40, 8, 32768, blocks=256, recent=16),
        # one ragged batch with few tokens: some sequences hold fewer blocks than are asked for
        _case("blocks ragged", "blocks", 5, 16, 2, 1999, page=64, ragged=True, dtype="f16", blocks=12, recent=1),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["append", "attend", "score", "blocks"])
    kv_heads = rng.choice([1, 2, 4, 8])
    head_dim = rng.choice([64, 128, 128, 256])
    page = rng.choice([16, 16, 32, 64, 128])
    batch = _log(rng, 1, 48)
    group = rng.choice([1, 2, 4, 5, 7, 8, 12])
    common = dict(head_dim=head_dim, page=page, ragged=rng.random() < 0.6, dtype=rng.choice(["bf16", "f16"]),
                  cache=rng.choice(["e4m3", "e4m3", "e5m2"]))
    width = batch * kv_heads * head_dim
    if op == "append":
        new = _log(rng, 1, max(2, min(20000, 33_000_000 // width)))
        tokens = rng.choice([0, _log(rng, 1, max(2, min(40000, 100_000_000 // width)))])
        if rng.random() < 0.25:
            common["dtype"] = "f32"
        return _case(None, op, batch, group * kv_heads, kv_heads, tokens, new=new, token_major=rng.random() < 0.5, **common)
    tokens = _log(rng, 1, min(131072, 500_000_000 // width))
    if op == "score":
        return _case(None, op, batch, group * kv_heads, kv_heads, tokens, **common)
    q_len = rng.choice([1, 1, 1, 2, 3, 5])
    if op == "attend":
        return _case(None, op, batch, group * kv_heads, kv_heads, max(1, tokens // q_len), q_len=q_len, **common)
    blocks = _log(rng, 1, max(2, min(512, 60_000_000 // (width * page))))
    return _case(None, op, batch, group * kv_heads, kv_heads, tokens, q_len=q_len, blocks=blocks,
                 recent=rng.choice([0, 1, 4]), **common)


def _lengths(case):
    """Tokens held by each sequence: all `tokens`, or spread from an eighth of them to all."""
    n, B = case["tokens"], case["batch"]
    if not case["ragged"] or n == 0:
        return [n] * B
    return [1 + (n - 1) * ((5 * b + 3) % 8 + 1) // 8 for b in range(B)]


def _news(case):
    """Tokens appended to each sequence."""
    n, B = case["new"], case["batch"]
    return [1 + (n - 1) * ((3 * b + 2) % 4 + 1) // 4 if case["ragged"] else n for b in range(B)]


def _pages_of(case, n):
    return -(-n // case["page"])


def _power(e):
    """2^e in 32 bits, exactly."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _encode(x, cache):
    """Codes and exponents of x [..., tokens, D], one exponent for each leading index."""
    a = x.abs().amax(dim=(-2, -1)).float()
    f, e = torch.frexp(a)
    # a = 2f * 2^(e-1); the largest code is 1.75 * 2^8 or 1.75 * 2^15
    e = e - 1 - (8 if cache == "e4m3" else 15) + (f > 0.875).to(e.dtype)
    e = torch.where(a == 0, torch.full_like(e, LOW), e).clamp(LOW, HIGH)
    y = x.float() * _power(-e)[..., None, None]
    return y.clamp(-LARGEST[cache], LARGEST[cache]).to(CACHE[cache]), e.to(torch.int8)


def prepare(case, seed):
    B, H, D, page = case["batch"], case["kv_heads"], case["head_dim"], case["page"]
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    lens, news = _lengths(case), _news(case)
    width = _pages_of(case, case["tokens"] + case["new"] + page)
    pages = B * width
    dtype = TYPES[case["dtype"]]
    # some channels of real keys are much larger than the others
    channel = torch.exp2(torch.randint(-1, 3, (H, 1, D), generator=g, device=dev).half())
    k, ke = _encode(torch.randn(pages, H, page, D, generator=g, device=dev, dtype=torch.float16) * channel, case["cache"])
    v, ve = _encode(torch.randn(pages, H, page, D, generator=g, device=dev, dtype=torch.float16), case["cache"])
    s = {"case": case, "k": k, "v": v, "exps": torch.stack([ke, ve], dim=-1).contiguous(),
         "table": torch.randperm(pages, generator=g, device=dev).to(torch.int32).view(B, width),
         "lens": torch.tensor(lens, dtype=torch.int32, device=dev)}
    f = k.to(torch.float16)
    s["bounds"] = torch.stack([f.amin(dim=2), f.amax(dim=2)], dim=2).to(CACHE[case["cache"]])
    del f
    if case["op"] == "append":
        n = case["new"]
        shape = (B, n, H, D) if case["token_major"] else (B, H, n, D)
        for name in ("k_new", "v_new"):
            x = torch.randn(shape, generator=g, device=dev, dtype=torch.float32).to(dtype)
            s[name] = x.transpose(1, 2) if case["token_major"] else x
        s["counts"] = torch.tensor(news, dtype=torch.int32, device=dev)
        return s
    s["q"] = torch.randn(B, case["q_heads"], case["q_len"], D, generator=g, device=dev, dtype=torch.float32).to(dtype)
    if case["op"] == "score":
        s["q"] = s["q"][:, :, 0].contiguous()
        s["out"] = torch.zeros(B, H, max(1, _pages_of(case, case["tokens"])), dtype=torch.float32, device=dev)
    if case["op"] == "blocks":
        held = (s["lens"].long() + page - 1) // page
        total = min(width, case["blocks"] + case["recent"])
        # random blocks and the last ones, in ascending order
        r = torch.rand(B, H, width, generator=g, device=dev)
        at = torch.arange(width, device=dev)
        r = r + (at >= (held - case["recent"])[:, None, None]).float()
        r = torch.where(at < held[:, None, None], r, torch.full_like(r, -1))
        best = r.topk(total, dim=-1).indices
        order = torch.where(best < held[:, None, None], best, best + width).sort(dim=-1).values
        s["blocks"] = torch.where(order < width, order, torch.zeros_like(order)).to(torch.int32)
        s["counts"] = held.clamp(max=total).to(torch.int32)[:, None].expand(B, H).contiguous()
    return s


def run(s):
    case = s["case"]
    if own:
        from mserve_b200 import ops
        pages = ops.Kv8Pages(s["k"], s["v"], s["exps"], s["bounds"])
        if case["op"] == "append":
            ops.kv8_append(pages, s["table"], s["k_new"], s["v_new"], tok0=s["lens"], counts=s["counts"])
            return s["k"], s["v"], s["exps"], s["bounds"]
        if case["op"] == "score":
            return ops.kv8_block_score(s["q"], pages, s["table"], lens=s["lens"], max_blocks=s["out"].shape[2], out=s["out"])
        if case["op"] == "blocks":
            return ops.kv8_attention(s["q"], pages, s["table"], lens=s["lens"], blocks=s["blocks"], counts=s["counts"])
        return ops.kv8_attention(s["q"], pages, s["table"], lens=s["lens"], max_tokens=case["tokens"])
    return {"append": _append, "score": _score, "attend": _attend, "blocks": _blocks}[case["op"]](s)


def _append(s):
    case, page = s["case"], s["case"]["page"]
    B, H, n, D = s["k_new"].shape
    tok0, counts = s["lens"].long(), s["counts"].long()
    touched = (n + page - 2) // page + 1                                         # pages a sequence can touch
    first = tok0 // page
    p = first[:, None] + torch.arange(touched, device=tok0.device)               # [B, touched]
    t = p[:, :, None] * page + torch.arange(page, device=tok0.device)            # [B, touched, page]
    old = t < tok0[:, None, None]
    fresh = (t >= tok0[:, None, None]) & (t < (tok0 + counts)[:, None, None])
    use = fresh.any(dim=-1)                                                      # [B, touched]
    p = p.clamp(max=s["table"].shape[1] - 1)
    at = s["table"].long().gather(1, p)                                          # physical pages
    src = (t - tok0[:, None, None]).clamp(0, n - 1)
    keep = use[:, :, None, None, None] & (old | fresh)[:, :, None, :, None]
    exps = s["exps"][at]                                                         # [B, touched, H, 2]
    for i, (pool, rows) in enumerate(((s["k"], s["k_new"]), (s["v"], s["v_new"]))):
        codes = pool[at]                                                         # [B, touched, H, page, D]
        x = codes.float() * _power(exps[..., i])[..., None, None]
        new = rows.float().transpose(1, 2)[torch.arange(B, device=at.device)[:, None, None], src]
        x = torch.where(fresh[:, :, None, :, None], new.transpose(2, 3), x)
        x = torch.where(keep, x, torch.zeros_like(x))
        q, e = _encode(x, case["cache"])
        pool[at] = torch.where(keep, q.float(), codes.float()).to(pool.dtype)
        exps[..., i] = torch.where(use[:, :, None], e, exps[..., i])
        if i == 0:
            valid = (old | fresh)[:, :, None, :, None]
            lo = torch.where(valid, q.float(), torch.full_like(x, math.inf)).amin(dim=3)
            hi = torch.where(valid, q.float(), torch.full_like(x, -math.inf)).amax(dim=3)
            both = torch.where(use[:, :, None, None, None], torch.stack([lo, hi], dim=3), s["bounds"][at].float())
            s["bounds"][at] = both.to(pool.dtype)
    s["exps"][at] = exps
    return s["k"], s["v"], s["exps"], s["bounds"]


def _score(s):
    q = s["q"].float()
    B, Hq, D = q.shape
    H, NB, page = s["k"].shape[1], s["out"].shape[2], s["case"]["page"]
    at = s["table"][:, :NB].long()
    b = s["bounds"][at].float()                                                  # [B, NB, H, 2, D]
    up = q.clamp(min=0).view(B, H, Hq // H, D).sum(dim=2)
    down = q.clamp(max=0).view(B, H, Hq // H, D).sum(dim=2)
    r = (b[..., 1, :] * up[:, None] + b[..., 0, :] * down[:, None]).sum(dim=-1)  # [B, NB, H]
    r = (r * _power(s["exps"][at][..., 0])).transpose(1, 2)
    held = (s["lens"].long() + page - 1) // page
    s["out"].copy_(torch.where(torch.arange(NB, device=r.device) < held[:, None, None], r, s["out"]))
    return s["out"]


def _softmax_product(q, k, v, visible):
    """q [B, H, G, Q, D], k and v [B, H, T, D], visible [B, 1 or H, Q, T]; rows that see nothing are zero."""
    B, H, G, Q, D = q.shape
    x = torch.matmul(q.float().reshape(B, H, G * Q, D), k.transpose(2, 3)) / math.sqrt(D)
    x = x.view(B, H, G, Q, -1).masked_fill(~visible[:, :, None], -math.inf)
    m = x.amax(dim=-1, keepdim=True)
    p = torch.exp(x - torch.where(m == -math.inf, torch.zeros_like(m), m))
    total = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p.view(B, H, G * Q, -1), v).view(B, H, G, Q, D)
    return torch.where(total > 0, o / total, torch.zeros_like(o))


def _attend(s):
    q, page = s["q"], s["case"]["page"]
    B, Hq, Q, D = q.shape
    H, T = s["k"].shape[1], s["case"]["tokens"]
    at = s["table"][:, :_pages_of(s["case"], T)].long()
    scale = _power(s["exps"][at])                                                # [B, pages, H, 2]
    t = torch.arange(at.shape[1] * page, device=q.device)
    inside = t < s["lens"][:, None]
    k = (s["k"][at].float() * scale[..., 0, None, None]).transpose(1, 2).reshape(B, H, -1, D)
    v = (s["v"][at].float() * scale[..., 1, None, None]).transpose(1, 2).reshape(B, H, -1, D)
    v = v.masked_fill(~inside[:, None, :, None], 0.0)
    limit = s["lens"][:, None] - Q + 1 + torch.arange(Q, device=q.device)        # [B, Q]
    o = _softmax_product(q.view(B, H, Hq // H, Q, D), k, v, (t < limit[:, :, None])[:, None])
    return o.reshape(B, Hq, Q, D).to(q.dtype)


def _blocks(s):
    q, page = s["q"], s["case"]["page"]
    B, Hq, Q, D = q.shape
    H, S = s["blocks"].shape[1:]
    blk = s["blocks"].long()
    at = s["table"].long()[:, None].expand(B, H, -1).gather(2, blk)              # [B, H, S] physical pages
    head = torch.arange(H, device=q.device)[:, None]
    scale = _power(s["exps"][at, head])                                          # [B, H, S, 2]
    t = blk[..., None] * page + torch.arange(page, device=q.device)              # [B, H, S, page]
    listed_ = (torch.arange(S, device=q.device) < s["counts"][..., None])[..., None]
    limit = s["lens"][:, None] - Q + 1 + torch.arange(Q, device=q.device)        # [B, Q]
    visible = (listed_[:, :, None] & (t[:, :, None] < limit[:, None, :, None, None])).reshape(B, H, Q, S * page)
    inside = (listed_ & (t < s["lens"][:, None, None, None])).reshape(B, H, S * page, 1)
    k = (s["k"][at, head].float() * scale[..., 0, None, None]).reshape(B, H, S * page, D)
    v = (s["v"][at, head].float() * scale[..., 1, None, None]).reshape(B, H, S * page, D)
    o = _softmax_product(q.view(B, H, Hq // H, Q, D), k, v.masked_fill(~inside, 0.0), visible)
    return o.reshape(B, Hq, Q, D).to(q.dtype)


def work(case):
    B, H, D, page, Q = case["batch"], case["kv_heads"], case["head_dim"], case["page"], case["q_len"]
    lens, news = _lengths(case), _news(case)
    size = 4 if case["dtype"] == "f32" else 2
    rows = B * case["q_heads"] * D * Q
    if case["op"] == "append":
        touched = sum((n0 + n - 1) // page - n0 // page + 1 for n0, n in zip(lens, news))
        values = 2 * sum(news) * H * D
        older = 2 * sum(n0 % page for n0 in lens) * H * D                        # read again: they share the page's scale
        return {"bytes": values * (size + 1) + older + touched * (H * (2 + 2 * D) + 4), "flops": 4 * (values + older)}
    blocks = [_pages_of(case, n) for n in lens]
    if case["op"] == "score":
        return {"bytes": sum(blocks) * (H * (2 * D + 1 + 4) + 4) + rows * 2, "flops": 4 * D * H * sum(blocks)}
    if case["op"] == "blocks":
        total = [min(case["blocks"] + case["recent"], n) for n in blocks]
        tokens = [min(n * page, length) for n, length in zip(total, lens)]
        listed_bytes = sum(total) * H * (2 + 4 + 4)
    else:
        tokens = lens
        listed_bytes = sum(blocks) * (2 * H + 4)
    return {"bytes": sum(tokens) * 2 * H * D + listed_bytes + 4 * rows,
            "flops": 4 * Q * case["q_heads"] * D * sum(tokens)}


# ---- the definition in 64 bits, sequence by sequence -------------------------------------------------------------
def _powers(device):
    """2^LOW .. 2^HIGH in 64 bits."""
    return torch.tensor([2.0 ** i for i in range(LOW, HIGH + 1)], dtype=torch.float64, device=device)


def _nearest_code(y, cache):
    """y rounded to the nearest 8-bit code, ties to even: mantissa bits 3 or 2, least normal exponent -6 or -14."""
    bits, least = (3, -6) if cache == "e4m3" else (2, -14)
    _, x = torch.frexp(y)                                                        # |y| in [2^(x-1), 2^x)
    step = _powers(y.device)[(x - 1).clamp(min=least, max=HIGH).long() - bits - LOW]
    return (torch.round(y / step) * step).clamp(-LARGEST[cache], LARGEST[cache])


def exact(case, seed):
    s = prepare(case, seed)
    H, D, page, Q = case["kv_heads"], case["head_dim"], case["page"], case["q_len"]
    lens, news, table = _lengths(case), _news(case), s["table"].cpu().long()
    powers = _powers(s["k"].device)
    scale = powers[s["exps"].long() - LOW]                                       # [pages, H, 2]
    if case["op"] == "append":
        k, v, bounds = s["k"].double(), s["v"].double(), s["bounds"].double()
        for b, (n0, n) in enumerate(zip(lens, news)):
            p0, p1 = n0 // page, (n0 + n - 1) // page + 1
            at = table[b, p0:p1].to(k.device)
            lo, hi = n0 - p0 * page, n0 - p0 * page + n
            for i, (pool, rows) in enumerate(((k, s["k_new"]), (v, s["v_new"]))):
                was = pool[at]                                                   # [pages, H, page, D]
                x = (was * scale[at][:, :, i, None, None]).transpose(0, 1).reshape(H, -1, D)
                x[:, lo:hi] = rows[b, :, :n].double()
                x[:, hi:] = 0
                x = x.view(H, p1 - p0, page, D)
                need = x.abs().amax(dim=(2, 3)) / LARGEST[case["cache"]]
                e = torch.searchsorted(powers, need.contiguous()).clamp(max=HIGH - LOW)
                code = _nearest_code(x / powers[e][:, :, None, None], case["cache"]).reshape(H, -1, D)
                if i == 0:
                    full = code.clone()
                    full[:, hi:] = math.inf
                    low = full.view(H, p1 - p0, page, D).amin(dim=2)
                    full[:, hi:] = -math.inf
                    top = full.view(H, p1 - p0, page, D).amax(dim=2)
                    bounds[at] = torch.stack([low, top], dim=2).transpose(0, 1)
                flat = was.transpose(0, 1).reshape(H, -1, D)
                flat[:, :hi] = code[:, :hi]
                pool[at] = flat.view(H, p1 - p0, page, D).transpose(0, 1)
        return k, v, None, bounds
    q, G = s["q"].double(), case["q_heads"] // H
    if case["op"] == "score":
        out = s["out"].double()
        for b, n in enumerate(lens):
            at = table[b, :_pages_of(case, n)].to(q.device)
            x, c = q[b].view(H, G, 1, D), s["bounds"][at].double().transpose(0, 1)[:, None] # [H, 1, blocks, 2, D]
            best = torch.zeros(H, at.shape[0], dtype=torch.float64, device=q.device)
            for j in range(G):
                best += torch.maximum(x[:, j:j + 1] * c[..., 0, :], x[:, j:j + 1] * c[..., 1, :]).sum(dim=-1)[:, 0]
            out[b, :, :at.shape[0]] = best * scale[at][:, :, 0].t()
        return out
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for b, n in enumerate(lens):
        for h in range(H):
            if case["op"] == "blocks":
                blk = s["blocks"][b, h, :int(s["counts"][b, h])].long()
            else:
                blk = torch.arange(_pages_of(case, n), device=q.device)
            at = table[b].to(q.device)[blk]
            t = (blk[:, None] * page + torch.arange(page, device=q.device)).view(-1)
            k = (s["k"][at, h].double() * scale[at, h, 0, None, None]).view(-1, D)[t < n]
            v = (s["v"][at, h].double() * scale[at, h, 1, None, None]).view(-1, D)[t < n]
            t = t[t < n]
            for i in range(Q):
                seen = int((t < n - Q + 1 + i).sum()) if case["op"] == "attend" else None
                kk, vv = (k[:seen], v[:seen]) if seen is not None else (k[t < n - Q + 1 + i], v[t < n - Q + 1 + i])
                if kk.shape[0]:
                    out[b, h * G:(h + 1) * G, i] = torch.softmax(q[b, h * G:(h + 1) * G, i] @ kk.t() / math.sqrt(D), dim=-1) @ vv
    return out
