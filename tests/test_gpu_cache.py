"""The paged 8-bit cache's kernels against their definitions in 64 bits."""
import math

import pytest
import torch

import cache_reference as ref
import ssa_amd
from conftest import has_gpu

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not has_gpu(), reason="needs a ROCm GPU")]

DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# ---------------------------------------------------------------------------- plan
def _check_plan(cached, new, width, free, free_count, ps, T, seed=0):
    g = _gen(seed)
    pages = len(free) + 1000
    table = torch.randint(0, pages, (len(cached), width), generator=g).int()
    want_table = table.tolist()
    want = ref.plan(cached, new, want_table, free, free_count, ps, T)
    # a table of longer rows, as a view
    wide = torch.full((len(cached), width + 3), -7, dtype=torch.int32, device=DEV)
    wide[:, :width] = table.to(DEV)
    p = ssa_amd.plan_pages(_i32(cached), _i32(new), wide[:, :width], _i32(free),
                           _i32([free_count]), page_size=ps, num_rows=T)
    got = (p.starts, p.lengths, p.slots, p.positions, p.requests, p.free_count, p.refused)
    for name, w, x in zip(("starts", "lengths", "slots", "positions", "requests", "free_count",
                           "refused"), want, got):
        assert x.flatten().tolist() == (w if isinstance(w, list) else [w]), name
    assert wide[:, :width].tolist() == want_table
    assert bool((wide[:, width:] == -7).all())


@pytest.mark.parametrize("ps", [32, 64, 128])
@pytest.mark.parametrize("R,rows,T", [(1, 1, 1), (1, 700, 703), (5, 40, 200), (257, 9, 2400),
                                      (1000, 70, 40000)])
def test_plan_matches(R, rows, T, ps):
    g = _gen(R)
    cached = torch.randint(0, 300, (R,), generator=g).tolist()
    new = torch.randint(0, rows + 1, (R,), generator=g).tolist()
    free = torch.randperm(3 * R + 600, generator=g).tolist()
    _check_plan(cached, new, 40, free, len(free), ps, T)


def test_plan_refusals_by_pages_rows_width_and_sign():
    free = list(range(50))
    # the third needs more pages than are left, the fourth none, the fifth one
    _check_plan([0, 60, 10, 5, 64], [64, 10, 200, 7, 1], 8, free, 3, 64, 400)
    # one whose table is full is passed over and its pages go to the next
    _check_plan([100, 0], [100, 100], 3, free, 2, 64, 300)
    # rows that end past the batch
    _check_plan([0, 0, 0], [10, 20, 1], 3, free, 50, 32, 30)
    _check_plan([0, 0, 0], [10, 20, 1], 3, free, 50, 32, 29)
    # negative lengths; nothing new; no rows at all
    _check_plan([-1, 5, 0], [3, -2, 4], 3, free, 50, 32, 20)
    _check_plan([0, 31, 32], [0, 0, 0], 3, free, 50, 32, 5)
    _check_plan([0, 31, 32], [0, 0, 0], 3, free, 50, 32, 0)
    # an empty free list
    _check_plan([0, 31], [1, 1], 3, [9], 0, 32, 2)


def test_plan_of_the_most_requests():
    g = _gen(4)
    cached = torch.randint(0, 90, (16384,), generator=g).tolist()
    new = torch.randint(0, 3, (16384,), generator=g).tolist()
    _check_plan(cached, new, 4, torch.randperm(9000, generator=g).tolist(), 5000, 32, 16000)


# ---------------------------------------------------------------------------- append
def _same_cache(cache, want, what=""):
    got = ref.Cache.of(cache)
    for name in ("k_scale", "v_scale", "k", "v", "bounds"):
        x, y = getattr(got, name), getattr(want, name)
        same = (x == y) | (x.isnan() & y.isnan())
        assert bool(same.all()), f"{what} {name}: {int((~same).sum())} differ"


def _random_cache(P, H, d, ps, seed, spread=3.0):
    """A cache of random codes with scales 2^-spread .. 2^spread apart."""
    c = ssa_amd.PagedKVCache(P, H, d, ps, device=DEV)
    g = _gen(seed)
    D = c.k_codes.shape[3]
    k = torch.randn(P, H, ps, D, generator=g) * 100
    v = torch.randn(P, H, D, ps, generator=g) * 100
    k[..., d:], v[:, :, d:] = 0, 0
    c.k_codes.copy_(k.clamp(-448, 448).to(ref_f8()))
    c.v_codes.copy_(v.clamp(-448, 448).to(ref_f8()))
    kf = c.k_codes.float()
    c.bounds.copy_(torch.stack([kf.amin(2), kf.amax(2)], 2).to(ref_f8()))
    for s in (c.k_scale, c.v_scale):
        s.copy_(torch.exp2(torch.round((torch.rand(P, H, generator=g) * 2 - 1) * spread) - 7))
    return c


def ref_f8():
    return torch.float8_e4m3fn


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("d,ps,H", [(64, 32, 2), (128, 64, 3), (96, 128, 1), (50, 64, 2),
                                    (1, 32, 1), (256, 128, 1), (129, 64, 2)])
def test_append_matches(dtype, d, ps, H):
    g = _gen(d)
    c = _random_cache(9, H, d, ps, d)
    want = ref.Cache.of(c)
    # whole pages, a page's start, its middle, its end, single tokens, rows that are skipped
    slots = ([2 * ps + i for i in range(2 * ps + 5)] + [-1, 9 * ps, 1 << 40]
             + [5 * ps + i for i in range(7, ps)] + [6 * ps + 3, 7 * ps, 8 * ps + ps - 1, -5]
             + [11 + i for i in range(6)])
    T = len(slots)
    k = torch.randn(T, H, d, generator=g) * torch.exp(2 * torch.randn(T, 1, 1, generator=g))
    v = torch.randn(T, H, d, generator=g) * torch.exp(2 * torch.randn(T, 1, 1, generator=g))
    k, v = k.to(dtype), v.to(dtype)
    # rows of a wider buffer, heads apart
    kv = torch.zeros(T, 2 * H + 1, d + 3, dtype=dtype)
    kv[:, :H, :d], kv[:, H:2 * H, :d] = k, v
    kv = kv.to(DEV)
    s = torch.tensor(slots, device=DEV)
    ssa_amd.cache_append(c, kv[:, :H, :d], kv[:, H:2 * H, :d], s)
    want.append(k, v, torch.tensor(slots))
    _same_cache(c, want)


@pytest.mark.parametrize("T", [1, 1500, 5000])
def test_append_of_long_calls(T):
    """Each of the windows in which runs are looked for."""
    g = _gen(T)
    c = ssa_amd.PagedKVCache(T // 64 + 40, 1, 64, 64, device=DEV)
    want = ref.Cache.of(c)
    # one long prompt that starts mid-page, then single tokens
    n = T - min(T - 1, 37)
    slots = [70 + i for i in range(n)]
    slots += [(70 + n) // 64 * 64 + 64 * (i + 1) + i % 64 for i in range(T - n)]
    slots = [s if s < c.num_pages * 64 else -1 for s in slots]
    k, v = torch.randn(T, 1, 64, generator=g), torch.randn(T, 1, 64, generator=g)
    ssa_amd.cache_append(c, k.to(DEV), v.to(DEV), torch.tensor(slots, device=DEV))
    want.append(k, v, torch.tensor(slots))
    _same_cache(c, want)


def test_append_token_by_token_grows_the_scale():
    """A page filled one token at a time, growing and shrinking: every code is
    rounded again each time its scale grows."""
    d, ps = 72, 32
    c = ssa_amd.PagedKVCache(2, 2, d, ps, device=DEV)
    want = ref.Cache.of(c)
    g = _gen(1)
    for i in range(ps + 3):
        size = 2.0 ** ((i * 7) % 23 - 11)
        k, v = torch.randn(1, 2, d, generator=g) * size, torch.randn(1, 2, d, generator=g) / size
        s = torch.tensor([i])
        ssa_amd.cache_append(c, k.to(DEV), v.to(DEV), s.to(DEV))
        want.append(k, v, s)
        _same_cache(c, want, f"token {i}")


def test_append_takes_a_shorter_prefix_again():
    """Rows written over a page's later tokens (rejected guesses): the tokens
    below stay, the scale does not shrink."""
    d, ps = 64, 64
    c = ssa_amd.PagedKVCache(1, 1, d, ps, device=DEV)
    want = ref.Cache.of(c)
    g = _gen(2)
    for lo, n, size in ((0, 40, 1.0), (25, 10, 0.1), (25, 39, 9.0), (0, 3, 0.01)):
        k, v = (torch.randn(n, 1, d, generator=g) * size for _ in range(2))
        s = torch.arange(lo, lo + n)
        ssa_amd.cache_append(c, k.to(DEV), v.to(DEV), s.to(DEV))
        want.append(k, v, s)
        _same_cache(c, want, f"rows {lo}+{n}")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_append_rounds_every_number(dtype):
    """All 2^16 bit patterns of a 16-bit type (a sweep of fp32), each row with
    its own page: codes, scales, and rows that are not finite."""
    if dtype == F32:
        x = torch.arange(1 << 16, dtype=torch.int64) * 65537 % (1 << 32)
        x = (x - (x >= 1 << 31).long() * (1 << 32)).to(torch.int32).view(F32)
    else:
        x = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(dtype)
    x = x.reshape(256, 1, 256)
    y = x.flip(0).contiguous()
    c = ssa_amd.PagedKVCache(256, 1, 256, 32, device=DEV)
    want = ref.Cache.of(c)
    s = torch.arange(256) * 32
    ssa_amd.cache_append(c, x.to(DEV), y.to(DEV), s.to(DEV))
    want.append(x, y, s)
    _same_cache(c, want)


def test_append_marks_rows_that_are_not_finite():
    """One bad number in a key or a value: that row and head alone, and the
    page's bounds, then and later."""
    c = ssa_amd.PagedKVCache(3, 2, 64, 32, device=DEV)
    want = ref.Cache.of(c)
    g = _gen(3)
    k, v = torch.randn(50, 2, 64, generator=g), torch.randn(50, 2, 64, generator=g)
    k[3, 0, 5], k[7, 1, 0], v[9, 0, 63], v[40, 1, 2] = math.nan, math.inf, -math.inf, 2.0 ** 120
    k[11, 0, 1] = -1.3e36                                  # just below 2^120
    s = torch.arange(50)
    ssa_amd.cache_append(c, k.to(DEV), v.to(DEV), s.to(DEV))
    want.append(k, v, s)
    _same_cache(c, want)
    k, v, s = k[20:30], v[20:30], torch.arange(50, 60)
    ssa_amd.cache_append(c, k.to(DEV), v.to(DEV), s.to(DEV))
    want.append(k, v, s)
    _same_cache(c, want, "later")
    assert bool(ref.Cache.of(c).bounds[1, 1].isnan().all())
    s = torch.arange(32, 42)                               # the page begun again
    ssa_amd.cache_append(c, k.to(DEV), v.to(DEV), s.to(DEV))
    want.append(k, v, s)
    _same_cache(c, want, "again")
    assert not bool(ref.Cache.of(c).bounds[1].isnan().any())


# ---------------------------------------------------------------------------- batches
def _batch(lens, new, ps, P, seed, *, extra=0, width=None):
    """Lists (table, starts, requests, positions) of requests with lens[r]
    tokens, the last new[r] of them this batch's rows."""
    perm = torch.randperm(P, generator=_gen(seed)).tolist()
    width = width or max(-(-n // ps) for n in lens) + 1
    table, starts, req, pos = [], [0], [], []
    for r, (L, n) in enumerate(zip(lens, new)):
        held = [perm.pop() for _ in range(-(-L // ps))]
        table.append(held + [-1] * (width - len(held)))
        starts.append(starts[-1] + n)
        req += [r] * n
        pos += list(range(L - n, L))
    return table, starts, req + [-1] * extra, pos + [-1] * extra


def _plan(b):
    return ssa_amd.PagePlan(*[_i32(x) for x in b])


def _queries(T, Hq, d, dtype, seed, strided=False):
    q = torch.randn(T, Hq, d, generator=_gen(seed)).to(dtype)
    if not strided:
        return q, q.to(DEV)
    wide = torch.zeros(T, Hq + 2, d + 5, dtype=dtype, device=DEV)
    wide[:, 1:Hq + 1, 3:d + 3] = q.to(DEV)
    return q, wide[:, 1:Hq + 1, 3:d + 3]


# ---------------------------------------------------------------------------- select
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("Hq,H,d,ps,top,first,recent", [
    (8, 2, 64, 32, 5, 1, 2), (4, 4, 128, 32, 3, 1, 2), (6, 1, 200, 32, 9, 0, 1),
    (5, 1, 33, 64, 4, 2, 1), (32, 1, 128, 32, 1, 0, 1)])
def test_select_matches(dtype, Hq, H, d, ps, top, first, recent):
    lens, new = [1, ps * 9 + 5, ps * 3, ps * 40 + 1], [1, 3, 2, 1]
    b = _batch(lens, new, ps, 80, d, extra=2)
    c = _random_cache(80, H, d, ps, d)
    q, qd = _queries(len(b[2]), Hq, d, dtype, 5, strided=True)
    got = ssa_amd.select_pages(qd, c, _plan(b), top, first=first, recent=recent)
    want = ref.select(q, ref.Cache.of(c), b[0], b[2], b[3], top, first, recent)
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("n_pages", [700, 5000])
def test_select_over_many_pages(n_pages):
    ps, d, H = 32, 64, 1
    b = _batch([n_pages * ps - 3], [1], ps, n_pages, 3)
    c = _random_cache(n_pages, H, d, ps, 3)
    q, qd = _queries(1, 4, d, BF16, 6)
    for top in (2, 40, n_pages - 1):
        got = ssa_amd.select_pages(qd, c, _plan(b), top, first=1, recent=1)
        want = ref.select(q, ref.Cache.of(c), b[0], b[2], b[3], top, 1, 1)
        assert torch.equal(got.cpu(), want), top


@pytest.mark.parametrize("rows", [1, 300])
def test_select_over_the_widest_table(rows):
    """16,384 pages a request (the same ones again and again), in both forms that
    take them."""
    ps, d, H, W = 32, 64, 1, 16384
    table = torch.randint(0, 900, (1, W), generator=_gen(rows))
    req, pos = [0] * rows, [W * ps - rows + i for i in range(rows)]
    c = _random_cache(900, H, d, ps, 3)
    q, qd = _queries(rows, 2, d, F16, 6)
    plan = _plan((table.tolist(), [0, rows], req, pos))
    got = ssa_amd.select_pages(qd, c, plan, 33, first=1, recent=2)
    few = [0, rows - 1]
    want = ref.select(q[few], ref.Cache.of(c), table.tolist(), [0, 0], [pos[i] for i in few],
                      33, 1, 2)
    assert torch.equal(got[few].cpu(), want[:len(few)])


def test_select_ties_missing_pages_and_nan():
    """Equal pages go to the lowest, absent pages come last, a page with a bad
    token first; a query that is NaN or zero takes the lowest pages."""
    ps, d, n = 32, 64, 300
    b = _batch([n * ps] * 3, [1, 1, 1], ps, 3 * n, 1)
    c = _random_cache(3 * n, 2, d, ps, 1)
    u = c.bounds.view(torch.uint8)
    u[:] = u[torch.randint(0, 4, (3 * n,), generator=_gen(0)).to(DEV)]     # four kinds of page
    c.k_scale[:] = c.k_scale[0]
    for r, p in ((0, 17), (0, 18), (1, 5), (2, 290)):
        b[0][r][p] = -1 if p != 5 else 3 * n
    c.bounds.view(torch.uint8)[b[0][0][200], 0] = 0x7f
    q, qd = _queries(3, 4, d, F32, 2)
    q[1, 1, 3], q[2, :2] = math.nan, 0.0
    qd = q.to(DEV)
    for top in (3, 60, 298):
        got = ssa_amd.select_pages(qd, c, _plan(b), top, first=1, recent=1)
        want = ref.select(q, ref.Cache.of(c), b[0], b[2], b[3], top, 1, 1)
        assert torch.equal(got.cpu(), want), top


# ---------------------------------------------------------------------------- attend
def _check_attend(c, b, q, qd, *, pages=None, scale=None, out=None):
    d = q.shape[2]
    got = ssa_amd.cached_attention(qd, c, _plan(b), scale=scale, out=out,
                                   pages=None if pages is None else pages.to(DEV))
    want, *sizes = ref.attend(q, ref.Cache.of(c), b[0], b[2], b[3],
                                     d ** -0.5 if scale is None else scale, pages)
    assert got.dtype == q.dtype and got.shape == q.shape
    keys = max(b[3] + [0]) + 1
    tol = ref.attend_tolerance(want, *sizes, q.dtype, keys, d)
    x = got.cpu().double()
    assert torch.equal(x.isnan(), want.isnan())
    ok = ((x - want).abs() <= tol) | want.isnan()
    assert bool(ok.all()), (f"{int((~ok).sum())} of {ok.numel()} beyond their tolerance, worst "
                            f"{float(((x - want).abs() / tol).nan_to_num().max()):.3g} times")
    return got


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("Hq,H,d,ps", [(2, 2, 64, 32), (8, 2, 128, 64), (16, 1, 96, 128),
                                       (20, 1, 128, 64), (5, 1, 250, 64), (4, 4, 17, 32),
                                       (64, 2, 64, 128), (34, 2, 256, 32)])
def test_attention_matches(dtype, Hq, H, d, ps):
    """Ragged batches: one token, full and part pages, a page's first token,
    requests without rows, several rows each, padding behind."""
    lens = [1, ps, ps + 1, 5, 2 * ps - 1, 7 * ps + 9, 3]
    new = [1, 1, 1, 0, 9, 4, 3]
    b = _batch(lens, new, ps, 40, d, extra=3)
    c = _random_cache(40, H, d, ps, d)
    q, qd = _queries(len(b[2]), Hq, d, dtype, 7, strided=True)
    got = _check_attend(c, b, q, qd)
    assert bool((got[-3:] == 0).all())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("T,L,Hq,H,d,ps", [(130, 130, 4, 1, 64, 64), (77, 500, 3, 3, 128, 32),
                                           (200, 261, 8, 1, 96, 128), (90, 90, 16, 1, 256, 64)])
def test_attention_over_prompts(dtype, T, L, Hq, H, d, ps):
    b = _batch([L, 40, L // 2], [T, 1, L // 2], ps, 60, d, extra=1)
    c = _random_cache(60, H, d, ps, d)
    q, qd = _queries(len(b[2]), Hq, d, dtype, 8)
    _check_attend(c, b, q, qd)


@pytest.mark.parametrize("dtype,d,ps", [(BF16, 128, 64), (F32, 64, 32), (F16, 80, 128)])
def test_attention_over_long_contexts(dtype, d, ps):
    """Keys in several parts, requests of very different lengths."""
    lens = [40 * ps + 7, 3, 25 * ps, 90 * ps + 1]
    b = _batch(lens, [1, 1, 1, 1], ps, 200, d)
    c = _random_cache(200, 2, d, ps, d)
    q, qd = _queries(4, 8, d, dtype, 9)
    _check_attend(c, b, q, qd)
    _check_attend(c, b, q, qd, scale=0.01)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("Hq,H,d,ps,top", [(8, 2, 128, 64, 5), (4, 4, 64, 32, 40),
                                           (32, 1, 96, 128, 3), (12, 2, 256, 32, 9)])
def test_attention_over_chosen_pages(dtype, Hq, H, d, ps, top):
    """Any order, gaps of -1, pages past the row's own and past the table."""
    lens = [45 * ps + 3, ps * 2, 1, 9 * ps + 1]
    b = _batch(lens, [3, 2, 1, 1], ps, 80, d, extra=1)
    c = _random_cache(80, H, d, ps, d)
    T = len(b[2])
    g = _gen(top)
    pages = torch.stack([torch.randperm(48, generator=g)[:top] for _ in range(T * H)])
    pages = pages.reshape(T, H, top).int()
    pages[torch.rand(T, H, top, generator=g) < 0.2] = -1
    pages[0, 0] = -1                                       # nothing at all
    q, qd = _queries(T, Hq, d, dtype, 10)
    got = _check_attend(c, b, q, qd, pages=pages)
    assert bool((got[0, :Hq // H] == 0).all())


def test_attention_skips_absent_pages_and_zeroes_rows_without_keys():
    ps, d = 32, 64
    b = _batch([5 * ps, 2 * ps], [2, 1], ps, 9, 1, extra=2)
    b[0][0][2], b[0][0][4] = -1, 9                         # gone, out of range
    b[0][1][0] = b[0][1][1] = -3
    c = _random_cache(9, 2, d, ps, 1)
    q, qd = _queries(5, 4, d, F32, 11)
    got = _check_attend(c, b, q, qd)
    assert bool((got[2:] == 0).all())


def test_attention_with_a_bad_token():
    """A NaN token makes the rows that see it NaN, in that head, and no other;
    codes left behind a request's end and unused table entries do nothing."""
    ps, d, H = 32, 64, 2
    c = _random_cache(12, H, d, ps, 2)
    b = _batch([70, 70], [40, 3], ps, 12, 2)
    g = _gen(4)
    k, v = torch.randn(1, H, d, generator=g), torch.randn(1, H, d, generator=g)
    k[0, 1, 3] = math.inf
    slot = b[0][0][1] * ps + 20                            # key 52 of request 0
    before = ref.Cache.of(c)
    ssa_amd.cache_append(c, k.to(DEV), v.to(DEV), torch.tensor([slot], device=DEV))
    before.append(k, v, torch.tensor([slot]))
    c.k_codes.view(torch.uint8)[b[0][1][2], :, 6:] = 0x7f  # behind key 69
    q, qd = _queries(43, 4, d, BF16, 12)
    got = _check_attend(c, b, q, qd)
    nan = got.isnan().any(-1).cpu()
    seen = torch.tensor([r == 0 and p >= 52 for r, p in zip(b[2], b[3])])
    assert torch.equal(nan[:, 2:].all(1), seen) and not bool(nan[:, :2].any())


def test_attention_with_scales_far_apart():
    """Pages of very large and very small numbers in one request."""
    ps, d = 32, 64
    c = _random_cache(20, 1, d, ps, 5)
    b = _batch([20 * ps], [4], ps, 20, 5)
    c.v_scale.copy_(torch.exp2(torch.linspace(-60, 60, 20).round()).reshape(20, 1))
    c.k_scale.copy_(torch.exp2(torch.linspace(-30, -6, 20).round()).reshape(20, 1))
    q, qd = _queries(4, 2, d, F32, 13)
    _check_attend(c, b, q, qd)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("lens,new", [([20 * 32], [4]), ([20 * 32], [100]), ([640] * 2, [1, 1])])
def test_attention_with_pages_of_zeros(dtype, lens, new):
    """Pages whose values are all zero have the smallest scale there is; beside large
    numbers, first, last and in between, they add nothing and lose nothing."""
    ps, d = 32, 64
    for size, zeros in ((40, (0, 7, 8, 19)), (-50, (3, 19)), (2, (0, 1, 2, 18, 19)), (6, (5,))):
        c = _random_cache(40, 1, d, ps, 5)
        b = _batch(lens, new, ps, 40, 5)
        c.v_scale.fill_(2.0 ** size)
        for r in range(len(lens)):
            for p in zeros:
                c.v_codes.view(torch.uint8)[b[0][r][p]] = 0
                c.v_scale[b[0][r][p]] = 2.0 ** -100
        q, qd = _queries(len(b[2]), 2, d, F32, 13)
        if dtype == F16 and size > 10:
            continue                                       # results beyond its range
        _check_attend(c, b, q.to(dtype), qd.to(dtype))


def test_attention_over_a_table_of_longer_rows():
    """Block tables as a view of wider rows."""
    ps, d = 32, 64
    b = _batch([100, 300, 77], [1, 60, 3], ps, 30, 1)
    c = _random_cache(30, 2, d, ps, 1)
    q, qd = _queries(64, 4, d, BF16, 2)
    want = _check_attend(c, b, q, qd)
    wide = torch.full((3, 64), 10 ** 6, dtype=torch.int32, device=DEV)
    w = len(b[0][0])
    wide[:, 3:3 + w] = _i32(b[0])
    plan = _plan(b)
    plan.block_table = wide[:, 3:3 + w]
    assert torch.equal(ssa_amd.cached_attention(qd, c, plan), want)
    assert torch.equal(ssa_amd.select_pages(qd, c, plan, 2), ssa_amd.select_pages(qd, c, _plan(b), 2))


def test_attention_writes_only_its_rows():
    """A given output of other strides; what lies around it stays."""
    ps, d = 64, 80
    b = _batch([100, 7], [3, 2], ps, 5, 6)
    c = _random_cache(5, 2, d, ps, 6)
    q, qd = _queries(5, 6, d, BF16, 14)
    wide = torch.full((7, 8, d + 9), 5.0, dtype=BF16, device=DEV)
    out = wide[1:6, 1:7, 4:d + 4]
    got = _check_attend(c, b, q, qd, out=out)
    assert got.data_ptr() == out.data_ptr()
    mask = torch.ones_like(wide, dtype=torch.bool)
    mask[1:6, 1:7, 4:d + 4] = False
    assert bool((wide[mask] == 5).all())


def test_empty_calls():
    c = ssa_amd.PagedKVCache(2, 1, 64, 32, device=DEV)
    p = ssa_amd.PagePlan(_i32([[0, 1]]), _i32([0, 0]), _i32([]), _i32([]))
    q = torch.empty(0, 4, 64, device=DEV)
    assert ssa_amd.cached_attention(q, c, p).shape == (0, 4, 64)
    assert ssa_amd.select_pages(q, c, p, 2).shape == (0, 1, 2)
    ssa_amd.cache_append(c, q[:, :1], q[:, :1], torch.empty(0, dtype=torch.int64, device=DEV))


def test_offsets_beyond_32_bits():
    """A cache of more than 2^32 code bytes: pages at its end."""
    H, d, ps = 8, 128, 64
    P = (1 << 32) // (H * d * ps) + 40
    c = ssa_amd.PagedKVCache(P, H, d, ps, device=DEV)
    small = ref.Cache(3, H, ps, d, d)
    g = _gen(9)
    k, v = torch.randn(150, H, d, generator=g), torch.randn(150, H, d, generator=g)
    s = torch.arange(150)
    ssa_amd.cache_append(c, k.to(DEV), v.to(DEV), s.to(DEV) + (P - 3) * ps)
    small.append(k, v, s)
    for name in ("k_codes", "bounds"):
        assert torch.equal(ref.numbers(getattr(c, name)[P - 3:]),
                           small.k if name == "k_codes" else small.bounds)
    assert torch.equal(ref.numbers(c.v_codes[P - 3:]).transpose(2, 3), small.v)
    assert not bool(c.k_codes[:1000].view(torch.uint8).any())
    plan = ssa_amd.PagePlan(_i32([[P - 3, P - 2, P - 1]]), _i32([0, 2]), _i32([0, 0]),
                            _i32([148, 149]))
    q = torch.randn(2, 16, d, generator=g)
    got = ssa_amd.cached_attention(q.to(DEV), c, plan).cpu().double()
    want, *sizes = ref.attend(q, small, [[0, 1, 2]], [0, 0], [148, 149], d ** -0.5)
    tol = ref.attend_tolerance(want, *sizes, F32, 150, d)
    assert bool(((got - want).abs() <= tol).all())
    got = ssa_amd.select_pages(q.to(DEV), c, plan, 2).cpu()
    assert torch.equal(got, ref.select(q, small, [[0, 1, 2]], [0, 0], [148, 149], 2, 1, 1))


# ---------------------------------------------------------------------------- forms
# Which kernel and how many chunks a call takes follows from T, R, heads, table width and
# page size; these reach the forms that the small cases above do not.
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("d,ps", [(64, 32), (128, 64), (200, 128)])
def test_attention_of_many_single_tokens(dtype, d, ps):
    """Units enough that each wave takes one of its own: 700 requests, 8 kv heads."""
    g = _gen(d)
    R = 700
    lens = torch.randint(1, 3 * ps, (R,), generator=g).tolist()
    new = [1] * R
    new[5], new[9] = 0, 3
    lens[9] += 3
    b = _batch(lens, new, ps, 3 * R, d, extra=1)
    c = _random_cache(3 * R, 8, d, ps, d)
    q, qd = _queries(len(b[2]), 8, d, dtype, 3)
    _check_attend(c, b, q, qd)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("Hq,H,d,ps", [(8, 8, 64, 32), (32, 8, 128, 64), (40, 2, 96, 128)])
def test_attention_over_chosen_pages_for_many_rows(dtype, Hq, H, d, ps):
    """Lists for rows enough to fill the chip, one wave a list."""
    T = 4096 // H + 40
    b = _batch([30 * ps + 5, 2 * ps + T], [40, T], ps, 100 + T // ps, d)
    rows = len(b[2])
    c = _random_cache(100 + T // ps, H, d, ps, d)
    g = _gen(d)
    pages = torch.stack([torch.randperm(12, generator=g)[:3] for _ in range(rows * H)])
    pages = pages.reshape(rows, H, 3).int()
    q, qd = _queries(rows, Hq, d, dtype, 4)
    _check_attend(c, b, q, qd, pages=pages)


@pytest.mark.parametrize("Hq,H,d,ps,top", [(4, 2, 64, 64, 20), (33, 1, 128, 64, 9)])
def test_attention_over_many_chosen_pages_of_a_prompt(Hq, H, d, ps, top):
    """More keys a row than a wave takes alone, but rows of one request side by side."""
    T = 2050 // H
    b = _batch([25 * ps + T, 7], [T, 1], ps, 27 + T // ps, d)
    c = _random_cache(27 + T // ps, H, d, ps, d)
    g = _gen(Hq)
    pages = torch.stack([torch.randperm(24, generator=g)[:top] for _ in range((T + 1) * H)])
    q, qd = _queries(T + 1, Hq, d, BF16, 4)
    _check_attend(c, b, q, qd, pages=pages.reshape(T + 1, H, top).int())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("Hq,H,d,ps", [(4, 4, 64, 32), (8, 2, 128, 64), (6, 1, 256, 128)])
def test_attention_of_a_prompt_behind_a_long_context(dtype, Hq, H, d, ps):
    """A prompt's keys in several chunks, single tokens with their own beside it, in
    one call; and pages missing in the middle."""
    lens = [70 * ps + 11, 33 * ps, 2, 50 * ps + 1]
    b = _batch(lens, [90, 1, 0, 3], ps, 200, d, extra=2)
    b[0][0][20] = b[0][3][7] = -1
    b[0][0][21] = 5000
    c = _random_cache(200, H, d, ps, d)
    q, qd = _queries(len(b[2]), Hq, d, dtype, 5, strided=True)
    got = _check_attend(c, b, q, qd)
    assert bool((got[-2:] == 0).all())


@pytest.mark.parametrize("scale", [-0.2, 0.0, 30.0])
def test_attention_scales(scale):
    """Negative, zero and large factors: the running maximum is the scaled scores'."""
    ps, d = 64, 64
    for new in ([1, 1], [100, 1]):
        b = _batch([150, 70], new, ps, 9, 1)
        c = _random_cache(9, 2, d, ps, 1)
        q, qd = _queries(len(b[2]), 4, d, F32, 6)
        _check_attend(c, b, q, qd, scale=scale)


def test_a_bad_token_in_a_prompt():
    """NaN and infinite tokens inside a prompt's own rows: causal rows before them and
    other heads stay finite, in every form."""
    ps, d, H = 32, 64, 2
    for dtype in (F32, BF16, F16):
        c = _random_cache(12, H, d, ps, 2)
        b = _batch([130, 60], [100, 2], ps, 12, 2)
        g = _gen(4)
        for key, bad in ((57, math.nan), (100, math.inf)):
            k, v = torch.randn(1, H, d, generator=g), torch.randn(1, H, d, generator=g)
            v[0, 0, 3] = bad
            s = torch.tensor([b[0][0][key // ps] * ps + key % ps], device=DEV)
            ssa_amd.cache_append(c, k.to(DEV), v.to(DEV), s)
        q, qd = _queries(102, 4, d, dtype, 12)
        got = _check_attend(c, b, q, qd)
        nan = got.isnan().any(-1).cpu()
        seen = torch.tensor([r == 0 and p >= 57 for r, p in zip(b[2], b[3])])
        assert torch.equal(nan[:, :2].all(1), seen) and not bool(nan[:, 2:].any())


def test_select_of_many_rows():
    """Rows enough for a wave each, beside requests without enough pages to choose."""
    ps, d, H = 32, 64, 4
    b = _batch([60 * ps + 3, 700, 9], [500, 60, 1], ps, 100, 1, extra=2)
    c = _random_cache(100, H, d, ps, 1)
    q, qd = _queries(len(b[2]), 8, d, BF16, 2)
    got = ssa_amd.select_pages(qd, c, _plan(b), 7, first=2, recent=2)
    assert torch.equal(got.cpu(), ref.select(q, ref.Cache.of(c), b[0], b[2], b[3], 7, 2, 2))


@pytest.mark.parametrize("rows", [255, 256, 257, 511, 512])
def test_select_at_the_bounds_of_its_forms(rows):
    """Rows times kv heads (1 and 4) and table widths on both sides of each rule."""
    ps, d = 32, 64
    for H, Hq, width in ((1, 2, None), (4, 4, None), (4, 4, 600)):
        b = _batch([40 * ps + 3, 700], [rows - 30, 30], ps, 70, rows, width=width)
        c = _random_cache(70, H, d, ps, rows)
        q, qd = _queries(rows, Hq, d, BF16, H)
        got = ssa_amd.select_pages(qd, c, _plan(b), 7, first=1, recent=2)
        assert torch.equal(got.cpu(), ref.select(q, ref.Cache.of(c), b[0], b[2], b[3], 7, 1, 2))


@pytest.mark.parametrize("R", [256, 257, 1024, 1025, 4096, 4097])
def test_plan_at_the_bounds_of_its_forms(R):
    g = _gen(R)
    cached = torch.randint(0, 70, (R,), generator=g).tolist()
    new = torch.randint(0, 4, (R,), generator=g).tolist()
    _check_plan(cached, new, 3, torch.randperm(2 * R, generator=g).tolist(), R // 3, 32, 2 * R)


# ---------------------------------------------------------------------------- as used
def _layer(**kw):
    a = dict(d_model=256, num_heads=8, num_kv_heads=2, num_neighbors=128, window_size=16,
             causal=True)
    torch.manual_seed(0)
    return ssa_amd.SparseAttention(ssa_amd.SSAConfig(**(a | kw))).to(DEV).eval()


@torch.no_grad()
@pytest.mark.parametrize("sparse", [False, True])
def test_layer_over_cached_tokens(sparse):
    """Prompts in chunks, then single tokens, by PageTable: each step's output
    is the layer's on what the cache then holds, in 64 bits."""
    attn = _layer()
    ps, H, kv, d = 32, attn.H, attn.n_kv, attn.d_head
    cache, table = attn.new_cache(40, ps), ssa_amd.PageTable(3, 20, 40, ps, device=DEV)
    lengths = [0, 0, 0]
    for step, new in enumerate([[60, 0, 33], [100, 7, 1], [1, 1, 1], [1, 0, 2], [300, 1, 0]]):
        T = sum(new) + 2
        x = torch.randn(T, 256, generator=_gen(step)).to(DEV)
        plan = table.plan(_i32(new), T)
        got = attn.forward_cached(x, cache, plan, sparse=sparse)
        lengths = [a + b for a, b in zip(lengths, new)]
        assert table.lengths.tolist() == lengths and plan.refused.item() == 0
        c = ref.Cache.of(cache)
        q = attn.Wq(x).view(T, H, d)
        rows = plan.block_table.tolist(), plan.requests.tolist(), plan.positions.tolist()
        pages = None
        if sparse:
            top, first, recent = attn.page_budget(ps)
            pages = ref.select(q, c, *rows, top, first, recent)
        want, *sizes = ref.attend(q, c, *rows, attn.scale, pages)
        tol = ref.attend_tolerance(want, *sizes, F32, max(lengths), d)
        W = attn.Wo.weight.double().cpu()
        want, tol = want.reshape(T, -1), tol.reshape(T, -1)
        # the output projection: H d products and sums in fp32
        off = tol @ W.abs().T + 2 * H * d * 2.0 ** -24 * (want.abs() @ W.abs().T) + 1e-30
        assert bool(((got.cpu().double() - want @ W.T).abs() <= off).all()), step
    table.release(torch.tensor([0, 2]))
    assert table.free_count.item() == 40 - (-(-lengths[1] // ps))


@torch.no_grad()
def test_model_steps_agree_with_one_pass():
    """A model's hidden states token by token and in one call over the whole
    prompt, all keys seen.  The two fill their caches with codes of other
    scales, so they agree to what 8 bits hold: each of a head's numbers within
    2^-4 of its value or of 2^-9 of its page's scale."""
    torch.manual_seed(3)
    cfg = ssa_amd.SSAConfig(d_model=128, num_heads=4, num_kv_heads=2, causal=True)
    model = ssa_amd.SparseTransformer(cfg, num_layers=2, vocab_size=50).to(DEV).eval()
    ids = torch.randint(0, 50, (70,), generator=_gen(1)).to(DEV)
    one, many = model.new_caches(4, 32), model.new_caches(4, 32)
    ta, tb = (ssa_amd.PageTable(1, 3, 4, 32, device=DEV) for _ in range(2))
    whole = model.forward_cached(ids, one, ta.plan(_i32([70]), 70), sparse=False)
    steps = [model.forward_cached(ids[i:i + 1], many, tb.plan(_i32([1]), 1), sparse=False)
             for i in range(70)]
    assert whole.shape == (70, 128) and bool(whole.isfinite().all())
    # layer 0's keys are the same numbers on both sides, rounded at most twice
    a, b = ref.Cache.of(one[0]), ref.Cache.of(many[0])
    assert torch.equal(a.k_scale[:3], b.k_scale[:3])
    x, y = a.k * a.k_scale[..., None, None], b.k * b.k_scale[..., None, None]
    assert bool(((x - y).abs() <= 2.0 ** -9 * a.k_scale[..., None, None]).all())
    err = (torch.cat(steps) - whole).norm() / whole.norm()
    assert float(err) < 2.0 ** -4


@torch.no_grad()
def test_captured_step_replays():
    """A whole step (plan, append, select, attend) in a HIP graph, replayed with
    new inputs, with eager calls and synchronizations between, and a second
    graph beside it: each replay is the eager step's result."""
    ps, H, Hq, d, R = 32, 2, 8, 64, 3

    def make():
        return ssa_amd.PagedKVCache(60, H, d, ps, device=DEV), ssa_amd.PageTable(
            R, 20, 60, ps, device=DEV)

    def step(cache, table, q, k, v, new):
        plan = table.plan(new, q.shape[0])
        ssa_amd.cache_append(cache, k, v, plan.slots)
        pages = ssa_amd.select_pages(q, cache, plan, 4, first=1, recent=2)
        return (ssa_amd.cached_attention(q, cache, plan, pages=pages),
                ssa_amd.cached_attention(q, cache, plan), plan.slots, pages)

    T = 2 * R
    eager, captured = make(), make()
    bufs = [torch.zeros(T, n, d, device=DEV, dtype=BF16) for n in (Hq, H, H)]
    new = _i32([2] * R)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*make(), *bufs, new)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):                                     # two that share no workspace
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs = step(*captured, *bufs, new)
        graphs.append((gr, outs))
    for i in range(30):
        fresh = [torch.randn(T, n, d, generator=_gen(100 * i + n)).to(DEV, BF16) for n in (Hq, H, H)]
        rows = _i32([2, i % 3, 1])
        want = step(*eager, *fresh, rows)
        for x, y in zip(bufs, fresh):
            x.copy_(y)
        new.copy_(rows)
        gr, outs = graphs[i % 2]
        gr.replay()
        if i % 4 == 0:
            torch.cuda.synchronize()
        for n, (x, y) in enumerate(zip(outs, want)):
            assert torch.equal(x, y), (i, n)
        assert torch.equal(captured[1].lengths, eager[1].lengths)
    _same_cache(captured[0], ref.Cache.of(eager[0]))


@torch.no_grad()
def test_captured_layer_step_reads_the_weights_themselves():
    """The first call of a layer under capture, its weights changed in place later and
    eager calls between the replays: each replay is the eager step of a layer with the
    weights of that moment."""
    T, R, ps = 6, 3, 32

    def make():
        attn = _layer()
        return attn, attn.new_cache(40, ps), ssa_amd.PageTable(R, 12, 40, ps, device=DEV)

    def step(attn, cache, table, x, new):
        return attn.forward_cached(x, cache, table.plan(new, T))

    x, new = torch.zeros(T, 256, device=DEV), _i32([2] * R)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*make(), x, new)                              # another layer of the same sizes
    torch.cuda.current_stream().wait_stream(side)
    captured, eager = make(), make()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = step(*captured, x, new)
    for i in range(12):
        if i % 3 == 2:
            for attn in (captured[0], eager[0]):
                for n, w in enumerate((attn.Wq, attn.Wk, attn.Wv, attn.Wo)):
                    w.weight.copy_(torch.randn(w.weight.shape, generator=_gen(9 * i + n)) / 16)
        x.copy_(torch.randn(T, 256, generator=_gen(i)))
        new.copy_(_i32([1, 2, i % 4]))
        want = step(*eager, x, new)
        torch.cuda.synchronize()
        gr.replay()
        junk = [torch.full((512, 256), float("nan"), device=DEV) for _ in range(4)]
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        del junk
    _same_cache(captured[1], ref.Cache.of(eager[1]))


def test_calls_on_another_stream():
    """Work queued on a side stream follows it."""
    ps, d = 64, 128
    b = _batch([3000, 900], [1, 1], ps, 64, 1)
    c = _random_cache(64, 2, d, ps, 1)
    q, qd = _queries(2, 8, d, BF16, 3)
    plan = _plan(b)
    want = ssa_amd.cached_attention(qd, c, plan)
    pages = ssa_amd.select_pages(qd, c, plan, 6)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        late = torch.zeros_like(qd)
        for _ in range(50):
            late.add_(1)
        late.copy_(qd)
        got = ssa_amd.cached_attention(late, c, plan)
        chosen = ssa_amd.select_pages(late, c, plan, 6)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(chosen, pages)


def test_repeated_calls_give_the_same_bits():
    ps, d = 64, 128
    b = _batch([9000, 4000, 100], [1, 1, 1], ps, 230, 1)
    c = _random_cache(230, 2, d, ps, 1)
    _, qd = _queries(3, 8, d, BF16, 3)
    first = ssa_amd.cached_attention(qd, c, _plan(b))
    for _ in range(5):
        assert torch.equal(ssa_amd.cached_attention(qd, c, _plan(b)), first)
