"""The serving operators over a paged 8-bit key/value cache, each in its plain form.

A cache page holds `page` tokens of every kv head as e4m3 codes, with one
power-of-two scale per page and head for the keys and one for the values:

    k_codes (pages, Hkv, page, D)    v_codes (pages, Hkv, D, page)
    k_scale, v_scale (pages, Hkv)    bounds (pages, Hkv, 2, D): per channel the
                                     smallest and the largest key code

D is the head dim rounded up to 64, 128 or 256.  A batch is ragged: request r
has its pages in `block_table[r]` and its new rows at `starts[r]` up to
`starts[r + 1]`; `requests` and `positions` say of every row whose it is and
where in its request it stands.  Four operators work on it:

    plan    block tables, slots, positions of a batch from its lengths
    append  the rows' keys and values into the cache
    select  for each row and kv head the pages that an upper bound of its
            scores ranks first, the first and the last ones always
    attend  softmax attention over all earlier keys, or over chosen pages

`own` False: elementary torch operations.  `own` True: ssa_amd's kernels.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
#: exponents of the scales, and the magnitude from which a number counts as not finite
E_MIN, E_MAX, TOO_BIG = -100, 112, 2.0 ** 120


# ---------------------------------------------------------------------------- cases
def _case(op, dtype, R, rows, lo, hi, Hq, Hkv, d, page, *, prompts=None, top=0):
    """R requests with lo..hi tokens before the call; the first `prompts` of
    them (all, if None) bring `rows` new rows each, the others one."""
    return dict(op=op, dtype=dtype, R=R, rows=rows, prompts=R if prompts is None else prompts,
                lo=lo, hi=hi, Hq=Hq, Hkv=Hkv, d=d, page=page, top=top)


def listed():
    return [
        # a small batch of single tokens: launches and host work count
        dict(_case("plan", "f32", 8, 1, 40, 4000, 8, 8, 64, 64), name="plan_few"),
        # a full server: a thousand requests, a tenth of them with prompts
        dict(_case("plan", "f32", 1000, 643, 1, 8191, 8, 8, 64, 64, prompts=100),
             name="plan_many"),
        # a decode step's keys and values into part-filled pages
        dict(_case("append", "bf16", 64, 1, 30, 8192, 32, 8, 128, 64), name="append_tokens_bf16"),
        # prompts of 2,731 tokens, head dim 96 stored as 128
        dict(_case("append", "f16", 3, 2731, 0, 100, 16, 8, 96, 128), name="append_prompt_f16"),
        # decode over long contexts: each token ranks its request's pages
        dict(_case("select", "bf16", 32, 1, 9000, 32767, 32, 8, 128, 64, top=32),
             name="select_tokens_bf16"),
        # a chunk of a long prompt, fp32
        dict(_case("select", "f32", 1, 1000, 15000, 15000, 16, 4, 64, 64, top=16),
             name="select_prompt_f32"),
        # the smallest attention call: two short fp32 requests
        dict(_case("attend", "f32", 2, 1, 90, 300, 8, 8, 64, 32), name="attend_tokens_f32"),
        # decode over long contexts, every key
        dict(_case("attend", "bf16", 16, 1, 5000, 32767, 32, 8, 128, 64),
             name="attend_tokens_bf16"),
        # prefill of 4,096 tokens
        dict(_case("attend", "bf16", 1, 4096, 0, 0, 32, 8, 128, 64), name="attend_prompt_bf16"),
        # one prompt's chunk among single tokens, ragged, fp16
        dict(_case("attend", "f16", 7, 777, 300, 2900, 16, 4, 64, 64, prompts=1),
             name="attend_mixed_f16"),
        # decode over 32 chosen pages of long contexts
        dict(_case("pages", "bf16", 32, 1, 9000, 32767, 32, 8, 128, 64, top=32),
             name="pages_tokens_bf16"),
        # a prompt's chunk, 16 pages a row
        dict(_case("pages", "bf16", 1, 1024, 8192, 8192, 32, 8, 128, 64, top=16),
             name="pages_prompt_bf16"),
    ]


def _span(rng, lo, hi):
    """A whole number of lo..hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "select", "attend", "attend", "pages"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    Hq, Hkv = rng.choice([(8, 8), (16, 16), (16, 4), (32, 8), (12, 4), (32, 1), (8, 2)])
    d = rng.choice([64, 128, 128, 96, 80, 32, 256])
    page = rng.choice([32, 64, 64, 128])
    if op == "plan":
        R = _span(rng, 1, 1000)
        return _case(op, dtype, R, _span(rng, 1, 640), rng.randint(0, 50), rng.randint(50, 8191),
                     Hq, Hkv, d, page, prompts=rng.randint(0, max(1, R // 10)))
    if op == "append":
        R = _span(rng, 1, 256)
        return _case(op, dtype, R, _span(rng, 1, max(2, 8000 // R)), rng.randint(0, 30),
                     rng.randint(30, 4000 if R > 64 else 16000), Hq, Hkv, min(d, 128), page)
    if rng.random() < 0.5:                                     # single tokens
        R, rows, hi = _span(rng, 1, 32), 1, _span(rng, 100, 32000)
    else:
        R, rows, hi = rng.randint(1, 4), _span(rng, 2, 900), _span(rng, 64, 8000)
    top = _span(rng, 3, 32) if op in ("select", "pages") else 0
    if op == "pages":                                          # gathered keys of the plain form
        while R * rows * Hkv * top * page * max(64, d) > 2.2e9:
            R, rows = max(1, R // 2), max(1, rows // 2)
    if op == "attend":                                         # scores and keys of the plain form
        while R * Hq * rows * (hi + rows) > 5e8 or R * Hkv * max(64, d) * hi > 5e8:
            hi, rows = hi // 2, max(1, rows * 3 // 4)
    return _case(op, dtype, R, rows, rng.randint(0, hi), hi, Hq, Hkv, d, page, top=top)


def _store(d):
    return 64 if d <= 64 else 128 if d <= 128 else 256


def _lengths(c):
    """(tokens before the call, new rows) of each request: the case's alone."""
    cached = [c["lo"] + int((c["hi"] - c["lo"]) * ((r * 0.6180339887498949) % 1.0))
              for r in range(c["R"])]
    new = [c["rows"] if r < c["prompts"] else 1 for r in range(c["R"])]
    return cached, new


def _forced(top):
    """(first, recent): a page of global tokens and the window's pages."""
    return 1, min(2, top - 1)


# ---------------------------------------------------------------------------- inputs
def _quantized(x, dim):
    """Codes of x with a power-of-two scale over `dim` (page-sized blocks)."""
    e = torch.ceil(torch.log2(x.abs().amax(dim, keepdim=True) / E4M3_MAX)).clamp_(E_MIN, E_MAX)
    s = torch.exp2(e)
    return (x / s).clamp_(-E4M3_MAX, E4M3_MAX).to(E4M3), s


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(DEV).manual_seed(seed)
    cached, new = _lengths(c)
    R, ps, H, d, D = c["R"], c["page"], c["Hkv"], c["d"], _store(c["d"])
    total = [a + b for a, b in zip(cached, new)]
    width = -(-max(total) // ps) + 1
    held = [-(-n // ps) for n in (cached if c["op"] == "plan" else total)]
    spare = sum(-(-n // ps) for n in total) - sum(held) + 5
    pages = sum(held) + spare
    perm = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    ids = torch.arange(width, device=DEV).expand(R, width)
    held_t = torch.tensor(held, device=DEV)
    first = torch.cumsum(held_t, 0) - held_t
    table = torch.where(ids < held_t[:, None], perm[(first[:, None] + ids).clamp(max=pages - 1)],
                        torch.full_like(ids, -1, dtype=torch.int32)).contiguous()
    T = sum(new)
    st = {"case": c, "table": table, "T": T, "max_new": max(new), "max_len": max(total)}
    cached_t = torch.tensor(cached, dtype=torch.int32, device=DEV)
    new_t = torch.tensor(new, dtype=torch.int32, device=DEV)
    if c["op"] == "plan":
        # a few rows of padding behind the last request, as a fixed-size batch has
        return st | {"cached": cached_t, "new": new_t, "T": T + 3, "free": perm[sum(held):].clone(),
                     "free_count": torch.tensor([spare], dtype=torch.int32, device=DEV)}
    starts = torch.zeros(R + 1, dtype=torch.int32, device=DEV)
    starts[1:] = torch.cumsum(new_t, 0)
    req = torch.repeat_interleave(torch.arange(R, device=DEV), new_t, output_size=T)
    row = torch.arange(T, device=DEV)
    pos = cached_t[req] + (row - starts[req])
    st |= {"starts": starts, "requests": req.to(torch.int32), "positions": pos.to(torch.int32)}
    dt = DTYPES[c["dtype"]]
    # channels of different size, as projected keys have
    chan = torch.exp(0.5 * torch.randn(H, 1, D, generator=g, device=DEV))
    chan[..., d:] = 0
    k = torch.randn(pages, H, ps, D, generator=g, device=DEV).mul_(chan)
    st["k_codes"], s = _quantized(k, (2, 3))
    st["k_scale"] = s.reshape(pages, H)
    del k
    v = torch.randn(pages, H, D, ps, generator=g, device=DEV)
    v[:, :, d:] = 0
    st["v_codes"], s = _quantized(v, (2, 3))
    st["v_scale"] = s.reshape(pages, H)
    del v
    kf = st["k_codes"].float()
    st["bounds"] = torch.stack([kf.amin(2), kf.amax(2)], 2).to(E4M3)
    del kf
    if c["op"] == "append":
        # the projections' output: keys and values side by side, 1 to 4 times the cached size
        kv = torch.randn(T, 2 * H, d, generator=g, device=DEV)
        kv *= torch.exp(1.4 * torch.rand(T, 1, 1, generator=g, device=DEV))
        kv = kv.to(dt)
        st["k"], st["v"] = kv[:, :H], kv[:, H:]
        st["slots"] = table[req, pos // ps].to(torch.int64) * ps + pos % ps
        return st
    st["q"] = torch.randn(T, c["Hq"], d, generator=g, device=DEV).to(dt)
    if c["op"] == "pages":
        # ascending distinct pages up to the row's own, -1 behind them
        top = c["top"]
        n = (pos // ps + 1)[:, None, None]
        r = torch.rand(T, H, width, generator=g, device=DEV)
        w = torch.arange(width, device=DEV)
        r = torch.where(w < n, torch.where((w == 0) | (w >= n - 2), r + 2, r), r - 4)
        ch = r.topk(min(top, width), -1).indices.sort(-1).values
        ch = torch.nn.functional.pad(ch, (0, top - ch.shape[-1]), value=width)
        ch, _ = torch.where(ch < n, ch, width).sort(-1)
        st["pages"] = torch.where(ch < n, ch, -1).to(torch.int32)
    return st


# ---------------------------------------------------------------------------- plain forms
def _plan(s):
    ps, T = s["case"]["page"], s["T"]
    cached, new, table = s["cached"].long(), s["new"].long(), s["table"]
    R, W = table.shape
    starts = torch.zeros(R + 1, dtype=torch.int64, device=DEV)
    starts[1:] = torch.cumsum(new, 0)
    had, want = (cached + ps - 1) // ps, (cached + new + ps - 1) // ps
    fits = (want <= W) & (starts[1:] <= T)
    need = torch.where(fits, want - had, 0)
    upto = torch.cumsum(need, 0)
    free = s["free_count"].long()
    ok = fits & ((need == 0) | (upto <= free))
    taken = torch.where(ok, need, 0).sum()
    col = torch.arange(W, device=DEV)
    k = (upto - need)[:, None] + col - had[:, None]
    fresh = ok[:, None] & (col >= had[:, None]) & (col < want[:, None])
    at = (free - 1 - k).clamp(0, s["free"].numel() - 1)
    table.copy_(torch.where(fresh, s["free"][at], table))
    row = torch.arange(T, device=DEV)
    req = torch.searchsorted(starts[1:].contiguous(), row, right=True)
    r = req.clamp(max=R - 1)
    live = (req < R) & ok[r]
    pos = cached[r] + row - starts[r]
    page = table[r, (pos // ps).clamp(0, W - 1)].long()
    return {"table": table, "starts": starts.int(),
            "lengths": torch.where(ok, cached + new, cached).int(),
            "slots": torch.where(live, page * ps + pos % ps, -1),
            "positions": torch.where(live, pos, -1).int(),
            "requests": torch.where(live, r, -1).int(),
            "free_count": (free - taken).int(), "refused": (~ok).sum(0, keepdim=True).int()}


def _append_half(x, codes, scale, page, off, pages, begun, transposed):
    """Rows x (T, H, D) into the touched pages of one of the two halves; the
    codes of those pages as numbers (n, H, ps, D) and which rows are written."""
    n, ps = pages.numel(), codes.shape[3 if transposed else 2]
    T, H, D = x.shape
    amax = torch.zeros(n, H, device=DEV).index_reduce_(0, page, x.abs().amax(2), "amax")
    e = torch.ceil(torch.log2(amax / E4M3_MAX)).clamp(E_MIN, E_MAX)
    e = torch.where(torch.exp2(e - 1) * E4M3_MAX >= amax, e - 1, e)      # log2 near a whole number
    e = torch.where(torch.exp2(e) * E4M3_MAX < amax, e + 1, e).clamp(E_MIN, E_MAX)
    old = torch.where(begun[:, None] > 0, scale[pages], torch.zeros_like(e))
    s = torch.maximum(old, torch.exp2(e))
    c = codes.view(torch.uint8)[pages].view(E4M3).float()
    c = c.transpose(2, 3) if transposed else c
    keep = (torch.arange(ps, device=DEV) < begun[:, None])[:, None, :, None]
    c = torch.where(keep, (c * (old / s)[:, :, None, None]).to(E4M3).float(), c)
    c = c.clone()
    c[page, :, off] = (x / s[page][:, :, None]).to(E4M3).float()
    out = (c.transpose(2, 3) if transposed else c).to(E4M3)
    codes.view(torch.uint8)[pages] = out.view(torch.uint8)
    scale[pages] = s
    return c, old / s


def _append(s):
    c = s["case"]
    ps, D = c["page"], s["k_codes"].shape[3]
    live = torch.nonzero(s["slots"] >= 0)[:, 0]
    slot = s["slots"][live]
    x, y = (torch.nn.functional.pad(t[live].float(), (0, D - c["d"])) for t in (s["k"], s["v"]))
    bad = ~((x.abs() < TOO_BIG).all(2) & (y.abs() < TOO_BIG).all(2))
    pages, page = torch.unique(slot // ps, return_inverse=True)
    off = slot % ps
    begun = torch.full((pages.numel(),), ps, device=DEV).index_reduce_(0, page, off, "amin")
    zero = torch.zeros((), device=DEV)
    x, y = torch.where(bad[:, :, None], zero, x), torch.where(bad[:, :, None], zero, y)
    k, shrink = _append_half(x, s["k_codes"], s["k_scale"], page, off, pages, begun, False)
    _append_half(y, s["v_codes"], s["v_scale"], page, off, pages, begun, True)
    k[page, :, off] = torch.where(bad[:, :, None], torch.full_like(zero, math.nan), k[page, :, off])
    s["k_codes"].view(torch.uint8)[pages] = k.to(E4M3).view(torch.uint8)
    b = s["bounds"].view(torch.uint8)[pages].view(E4M3).float()
    b = (b * shrink[:, :, None, None]).to(E4M3).float()
    was = (begun > 0)[:, None, None]
    inf = torch.full_like(zero, math.inf)
    new = torch.zeros(pages.numel(), ps, dtype=torch.bool, device=DEV)
    new[page, off] = True
    new = new[:, None, :, None]
    lo = torch.minimum(torch.where(was, b[:, :, 0], inf), torch.where(new, k, inf).amin(2))
    hi = torch.maximum(torch.where(was, b[:, :, 1], -inf), torch.where(new, k, -inf).amax(2))
    s["bounds"].view(torch.uint8)[pages] = torch.stack([lo, hi], 2).to(E4M3).view(torch.uint8)
    return {n: s[n] for n in ("k_codes", "v_codes", "bounds", "k_scale", "v_scale")}


def _select(s):
    c = s["case"]
    H, ps, top = c["Hkv"], c["page"], c["top"]
    first, recent = _forced(top)
    T, Hq, d = s["q"].shape
    R = s["table"].shape[0]
    W = -(-s["max_len"] // ps)
    bt = s["table"][:, :W].long().clamp(min=0)
    # 64 bits: which of two pages comes first is the formula's answer, not the sum's order
    b = s["bounds"].view(torch.uint8)[bt].view(E4M3).double()[..., :d]
    b = b * s["k_scale"][bt].double()[..., None, None]                     # (R, W, H, 2, d)
    q = s["q"].double().reshape(T, H, Hq // H, d)
    qq = torch.cat([q.clamp(min=0).sum(2), q.clamp(max=0).sum(2)], -1)      # (T, H, 2d)
    bb = torch.cat([b[:, :, :, 1], b[:, :, :, 0]], -1).permute(2, 3, 0, 1).reshape(H, 2 * d, R * W)
    sc = torch.matmul(qq.transpose(0, 1).contiguous(), bb.contiguous())     # (H, T, R W)
    req = s["requests"].long()
    sc = sc.reshape(H, T, R, W)[:, torch.arange(T, device=DEV), req].transpose(0, 1)
    n = (s["positions"].long() // ps + 1)[:, None, None]
    w = torch.arange(W, device=DEV)
    sc = torch.where(sc.isnan() | (w < first) | (w >= n - recent), math.inf, sc)
    # own pages before equal scores elsewhere, the lowest of equals first
    key = torch.where(w < n, sc, -math.inf)
    forced = ((w < first) | (w >= n - recent)) & (w < n)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    later = (~forced).expand_as(key).gather(-1, order).int()
    order = order.gather(-1, torch.sort(later, dim=-1, stable=True).indices)
    order = torch.nn.functional.pad(order, (0, max(0, top - W)), value=W)[..., :top]
    order = torch.where(order < n, order, W).sort(-1).values
    return torch.where(order < n, order, -1).int()


def _softmax_out(sc, seen, v):
    """softmax over the last axis of sc where seen, times v; nothing seen gives zeros."""
    sc = torch.where(seen, sc, -math.inf)
    m = sc.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(sc - torch.where(m == -math.inf, 0.0, m)), 0.0)
    tot = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(tot == 0, 1.0, tot)


def _attend(s):
    c = s["case"]
    H, ps = c["Hkv"], c["page"]
    T, Hq, d = s["q"].shape
    rep, n = Hq // H, s["max_new"]
    R = s["table"].shape[0]
    W = -(-s["max_len"] // ps)
    bt = s["table"][:, :W].long().clamp(min=0)
    k = s["k_codes"].view(torch.uint8)[bt].view(E4M3).float()[..., :d]
    k = (k * s["k_scale"][bt][..., None, None]).transpose(1, 2).reshape(R, H, W * ps, d)
    v = s["v_codes"].view(torch.uint8)[bt].view(E4M3).float()[:, :, :, :d]
    v = (v * s["v_scale"][bt][..., None, None]).permute(0, 2, 1, 4, 3).reshape(R, H, W * ps, d)
    starts = s["starts"].long()
    i = torch.arange(n, device=DEV)
    row = (starts[:-1, None] + i).clamp(max=T - 1)                          # (R, n)
    live = i < (starts[1:] - starts[:-1])[:, None]
    q = s["q"].float()[row].reshape(R, n, H, rep, d).permute(0, 2, 3, 1, 4).reshape(R, H, rep * n, d)
    sc = torch.matmul(q, k.transpose(2, 3)) * d ** -0.5
    pos = torch.where(live, s["positions"].long()[row], -1)
    seen = torch.arange(W * ps, device=DEV) <= pos[:, None, None, :, None]   # (R, 1, 1, n, keys)
    seen = seen.expand(R, 1, rep, n, W * ps).reshape(R, 1, rep * n, W * ps)
    o = _softmax_out(sc, seen, v).reshape(R, H, rep, n, d).permute(0, 3, 1, 2, 4)
    out = torch.zeros(T, Hq, d, device=DEV)
    out[row[live]] = o.reshape(R, n, Hq, d)[live]
    return out.to(s["q"].dtype)


def _attend_pages(s):
    c = s["case"]
    H, ps, K = c["Hkv"], c["page"], c["top"]
    T, Hq, d = s["q"].shape
    pages = s["pages"].long()
    phys = s["table"].long()[s["requests"].long()[:, None, None], pages.clamp(min=0)].clamp(min=0)
    h = torch.arange(H, device=DEV)[None, :, None]
    k = s["k_codes"].view(torch.uint8)[phys, h].view(E4M3).float()[..., :d]
    k = (k * s["k_scale"][phys, h][..., None, None]).reshape(T, H, K * ps, d)
    q = s["q"].float().reshape(T, H, Hq // H, d)
    sc = torch.matmul(q, k.transpose(2, 3)) * d ** -0.5
    v = s["v_codes"].view(torch.uint8)[phys, h].view(E4M3).float()[:, :, :, :d]
    v = (v * s["v_scale"][phys, h][..., None, None]).transpose(3, 4).reshape(T, H, K * ps, d)
    key = pages[..., None] * ps + torch.arange(ps, device=DEV)
    seen = (pages[..., None] >= 0) & (key <= s["positions"].long()[:, None, None, None])
    o = _softmax_out(sc, seen.reshape(T, H, 1, K * ps), v)
    return o.reshape(T, Hq, d).to(s["q"].dtype)


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        import ssa_amd
        if op == "plan":
            p = ssa_amd.plan_pages(s["cached"], s["new"], s["table"], s["free"], s["free_count"],
                                   page_size=s["case"]["page"], num_rows=s["T"])
            return {"table": p.block_table, "starts": p.starts, "lengths": p.lengths,
                    "slots": p.slots, "positions": p.positions, "requests": p.requests,
                    "free_count": p.free_count, "refused": p.refused}
        cache = ssa_amd.PagedKVCache.from_tensors(s["k_codes"], s["v_codes"], s["bounds"],
                                                  s["k_scale"], s["v_scale"], s["case"]["d"])
        if op == "append":
            ssa_amd.cache_append(cache, s["k"], s["v"], s["slots"])
            return {n: s[n] for n in ("k_codes", "v_codes", "bounds", "k_scale", "v_scale")}
        plan = ssa_amd.PagePlan(s["table"], s["starts"], s["requests"], s["positions"])
        if op == "select":
            first, recent = _forced(s["case"]["top"])
            return ssa_amd.select_pages(s["q"], cache, plan, s["case"]["top"], first=first,
                                        recent=recent)
        return ssa_amd.cached_attention(s["q"], cache, plan, pages=s.get("pages"))
    return {"plan": _plan, "append": _append, "select": _select, "attend": _attend,
            "pages": _attend_pages}[op](s)


# ---------------------------------------------------------------------------- work
def work(case):
    c = case
    cached, new = _lengths(c)
    ps, H, Hq, d, R, T = c["page"], c["Hkv"], c["Hq"], c["d"], c["R"], sum(new)
    es = 4 if c["dtype"] == "f32" else 2
    had = [-(-a // ps) for a in cached]
    want = [-(-(a + b) // ps) for a, b in zip(cached, new)]
    if c["op"] == "plan":
        taken = sum(want) - sum(had)
        return {"bytes": 16 * R + 8 * taken + 4 * R + 16 * T, "flops": 0}
    if c["op"] == "append":
        touched = sum(w - a // ps for w, a in zip(want, cached))
        return {"bytes": 2 * T * H * d * (es + 1) + 8 * T + touched * H * (4 * d + 16),
                "flops": 4 * T * H * d}
    qo = T * Hq * d * es
    if c["op"] == "select":
        n = sum(b * w for b, w in zip(new, want))
        return {"bytes": qo + sum(want) * H * (2 * d + 4) + 4 * T * H * c["top"],
                "flops": 4 * n * H * d}
    if c["op"] == "attend":
        keys = sum(b * a + b * (b + 1) // 2 for a, b in zip(cached, new))
        return {"bytes": 2 * qo + sum((a + b) * 2 * H * d for a, b in zip(cached, new)),
                "flops": 4 * keys * Hq * d}
    top = [min(c["top"], w) for w in want]
    keys = sum(b * min(t * ps, a + 1) for t, a, b in zip(top, cached, new))
    read = sum(min(b * t, w) * ps for b, t, w in zip(new, top, want))
    return {"bytes": 2 * qo + 2 * read * H * d + 4 * T * H * c["top"], "flops": 4 * keys * Hq * d}


# ---------------------------------------------------------------------------- 64-bit results
def _values():
    """The number each of the 256 codes stands for: sign, 4 exponent bits
    (bias 7), 3 mantissa bits; all ones but the sign is NaN."""
    t = []
    for b in range(256):
        e, m = (b >> 3) & 15, b & 7
        v = math.nan if b & 127 == 127 else (math.ldexp(m, -9) if e == 0
                                             else math.ldexp(8 + m, e - 10))
        t.append(-v if b & 128 else v)
    return torch.tensor(t, dtype=torch.float64, device=DEV)


def _to_code(x):
    """The code value nearest to x (|x| <= 448), ties to the even mantissa."""
    _, e = torch.frexp(x)
    step = torch.exp2((e.double() - 1).clamp(min=-6) - 3)
    return torch.round(x / step) * step


def _exact_append(s):
    c, val = s["case"], _values()
    ps, d = c["page"], c["d"]
    out = {n: val[s[n].view(torch.uint8).long()] for n in ("k_codes", "v_codes", "bounds")}
    out |= {n: s[n].double() for n in ("k_scale", "v_scale")}
    k, v = out["k_codes"], out["v_codes"].transpose(2, 3)
    slots = s["slots"].tolist()
    t = 0
    while t < len(slots):
        n = 1
        while t + n < len(slots) and slots[t + n] == slots[t] + n and slots[t + n] % ps:
            n += 1
        p, o = divmod(slots[t], ps)
        for name, dst, src in (("k", k, s["k"]), ("v", v, s["v"])):
            x = src[t:t + n].double().transpose(0, 1)                       # (H, n, d)
            a = x.abs().amax((1, 2))
            m, e = torch.frexp(a / 448.0)
            e = torch.where(m == 0.5, e - 1, e).clamp(E_MIN, E_MAX)         # 2^e >= a / 448
            e = torch.where(a == 0, E_MIN, e)
            sc = torch.exp2(e.double())
            if o:
                sc = torch.maximum(sc, out[name + "_scale"][p])
                ratio = out[name + "_scale"][p] / sc
                dst[p, :, :o] = _to_code(dst[p, :, :o] * ratio[:, None, None])
                if name == "k":
                    out["bounds"][p] = _to_code(out["bounds"][p] * ratio[:, None, None])
            out[name + "_scale"][p] = sc
            dst[p, :, o:o + n, :d] = _to_code(x / sc[:, None, None])
            dst[p, :, o:o + n, d:] = 0
            if name == "k":
                q = dst[p, :, o:o + n]
                q = torch.stack([q.amin(1), q.amax(1)], 1)
                b = out["bounds"][p]
                out["bounds"][p] = q if not o else torch.stack(
                    [torch.minimum(b[:, 0], q[:, 0]), torch.maximum(b[:, 1], q[:, 1])], 1)
        t += n
    return out


def _exact_attend(s):
    c, val = s["case"], _values()
    H, ps = c["Hkv"], c["page"]
    T, Hq, d = s["q"].shape
    out = torch.zeros(T, Hq, d, dtype=torch.float64, device=DEV)
    cached, new = _lengths(c)
    t = 0
    for r, (a, n) in enumerate(zip(cached, new)):
        p = s["table"][r, :-(-(a + n) // ps)].long()
        pos = torch.arange(a, a + n, device=DEV)[:, None]
        j = torch.arange(p.numel() * ps, device=DEV)
        for h in range(H):
            k = val[s["k_codes"][p, h].view(torch.uint8).long()] * s["k_scale"][p, h][:, None, None]
            v = val[s["v_codes"][p, h].view(torch.uint8).long()] * s["v_scale"][p, h][:, None, None]
            k, v = k.reshape(-1, k.shape[-1])[:, :d], v.transpose(1, 2).reshape(-1, k.shape[-1])[:, :d]
            seen = j <= pos
            if c["op"] == "pages":
                ch = s["pages"][t:t + n, h].long()
                hit = torch.zeros(n, p.numel() + 1, dtype=torch.bool, device=DEV)
                hit.scatter_(1, torch.where(ch < 0, p.numel(), ch), True)
                seen = seen & hit[:, :-1].repeat_interleave(ps, 1)
            for g in range(h * (Hq // H), (h + 1) * (Hq // H)):
                z = torch.where(seen, s["q"][t:t + n, g].double() @ k.T * d ** -0.5, -math.inf)
                z = torch.exp(z - z.amax(1, keepdim=True))
                out[t:t + n, g] = (z @ v) / z.sum(1, keepdim=True)
        t += n
    return out


def exact(case, seed):
    if case["op"] in ("plan", "select"):
        return None                                            # whole numbers only
    s = prepare(case, seed)
    return _exact_append(s) if case["op"] == "append" else _exact_attend(s)
