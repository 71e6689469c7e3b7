"""The paged 8-bit cache's operators in 64 bits, on the CPU, written from their
definitions (test infrastructure)."""
import math

import torch

E_MIN, E_MAX, TOO_BIG = -100, 112, 2.0 ** 120


def _values():
    t = []
    for b in range(256):
        e, m = (b >> 3) & 15, b & 7
        v = math.nan if b & 127 == 127 else (math.ldexp(m, -9) if e == 0
                                             else math.ldexp(8 + m, e - 10))
        t.append(-v if b & 128 else v)
    return torch.tensor(t, dtype=torch.float64)


VALUES = _values()


def numbers(codes):
    """The numbers a tensor of e4m3 codes stands for."""
    return VALUES[codes.cpu().view(torch.uint8).long()]


def to_code(x):
    """The e4m3 number nearest to x (|x| <= 448), ties to the even mantissa."""
    _, e = torch.frexp(x)
    step = torch.exp2((e.double() - 1).clamp(min=-6) - 3)
    return torch.round(x / step) * step


def exponent(a):
    """Smallest e in E_MIN..E_MAX with a <= 448 * 2^e."""
    e = E_MIN
    while e < E_MAX and a > math.ldexp(448.0, e):
        e += 1
    return e


class Cache:
    """Numbers, not codes: k, v (pages, H, page, D), bounds (pages, H, 2, D)."""

    def __init__(self, pages, H, ps, D, d):
        self.ps, self.D, self.d = ps, D, d
        self.k = torch.zeros(pages, H, ps, D, dtype=torch.float64)
        self.v = torch.zeros(pages, H, ps, D, dtype=torch.float64)
        self.bounds = torch.zeros(pages, H, 2, D, dtype=torch.float64)
        self.k_scale = torch.ones(pages, H, dtype=torch.float64)
        self.v_scale = torch.ones(pages, H, dtype=torch.float64)

    @classmethod
    def of(cls, cache):
        """The numbers of a PagedKVCache as it stands."""
        P, H, ps, D = cache.k_codes.shape
        self = cls(P, H, ps, D, cache.d_head)
        self.k, self.v = numbers(cache.k_codes), numbers(cache.v_codes).transpose(2, 3)
        self.bounds = numbers(cache.bounds)
        self.k_scale, self.v_scale = cache.k_scale.cpu().double(), cache.v_scale.cpu().double()
        return self

    def append(self, k, v, slots):
        k, v = k.cpu().double(), v.cpu().double()
        P, H = self.k_scale.shape
        slots = slots.tolist()
        t = 0
        while t < len(slots):
            n = 1
            while (t + n < len(slots) and slots[t + n] == slots[t] + n
                   and slots[t + n] % self.ps):
                n += 1
            if 0 <= slots[t] < P * self.ps:
                p, o = divmod(slots[t], self.ps)
                for h in range(H):
                    self._rows(p, h, o, k[t:t + n, h], v[t:t + n, h])
            t += n

    def _rows(self, p, h, o, x, y):
        n = x.shape[0]
        bad = ~((x.abs() < TOO_BIG).all(1) & (y.abs() < TOO_BIG).all(1))
        for rows, dst, scale, src in ((self.k, self.k[p, h], self.k_scale, x),
                                      (self.v, self.v[p, h], self.v_scale, y)):
            src = torch.where(bad[:, None], 0.0, src)
            s = math.ldexp(1.0, exponent(float(src.abs().max())))
            if o:
                s = max(s, float(scale[p, h]))
                r = float(scale[p, h]) / s
                dst[:o] = to_code(dst[:o] * r)
                if rows is self.k:
                    self.bounds[p, h] = to_code(self.bounds[p, h] * r)
            scale[p, h] = s
            dst[o:o + n] = 0
            dst[o:o + n, :self.d] = to_code(src / s)
        self.k[p, h, o:o + n][bad] = math.nan
        c = self.k[p, h, o:o + n]
        lo, hi = c.amin(0), c.amax(0)
        if o:
            lo, hi = torch.minimum(lo, self.bounds[p, h, 0]), torch.maximum(hi, self.bounds[p, h, 1])
        if bad.any():
            lo, hi = torch.full_like(lo, math.nan), torch.full_like(hi, math.nan)
        self.bounds[p, h, 0], self.bounds[p, h, 1] = lo, hi


def plan(cached, new, table, free, free_count, ps, T):
    """(starts, lengths, slots, positions, requests, free_count, refused); the
    table (a list of lists) takes the new pages."""
    starts, lengths = [0], []
    slots, positions, requests = [-1] * T, [-1] * T, [-1] * T
    asked, taken, refused = 0, 0, 0
    for r, (c, n) in enumerate(zip(cached, new)):
        s = starts[-1]
        starts.append(s + max(n, 0))
        want, had = -(-(c + n) // ps), -(-c // ps)
        ok = c >= 0 and n >= 0 and want <= len(table[r]) and starts[-1] <= T
        if ok:
            asked += want - had
            ok = want == had or asked <= free_count
        if not ok:
            refused += 1
            lengths.append(c)
            continue
        for col in range(had, want):
            table[r][col] = free[free_count - 1 - taken]
            taken += 1
        lengths.append(c + n)
        for i in range(n):
            page = table[r][(c + i) // ps]
            slots[s + i] = page * ps + (c + i) % ps if page >= 0 else -1
            positions[s + i], requests[s + i] = c + i, r
    return starts, lengths, slots, positions, requests, free_count - taken, refused


def select(q, c, table, requests, positions, top, first, recent):
    """Page lists as nested Python lists (T, H, top)."""
    T, Hq, d = q.shape
    P, H = c.k_scale.shape
    q = q.cpu().double().reshape(T, H, Hq // H, d)
    out = torch.full((T, H, top), -1, dtype=torch.int32)
    for t in range(T):
        r, pos = requests[t], positions[t]
        if r < 0 or r >= len(table) or pos < 0:
            continue
        n = min(pos // c.ps + 1, len(table[r]))
        for h in range(H):
            if n <= top:
                out[t, h, :n] = torch.arange(n)
                continue
            cand = []
            for p in range(first, n - recent):
                pg = table[r][p]
                if not 0 <= pg < P:
                    cand.append((2, 0.0, p))
                    continue
                # the channel sums of the formula, exact products in 64 bits
                qp, qm = q[t, h].clamp(min=0).sum(0), q[t, h].clamp(max=0).sum(0)
                b = c.bounds[pg, h, :, :d]
                s = float(((qm * b[0]).sum() + (qp * b[1]).sum()) * c.k_scale[pg, h])
                cand.append((1, -math.inf if math.isnan(s) else -s, p))
            best = sorted(cand)[:top - first - recent]
            pick = sorted([p for _, _, p in best] + list(range(first)) + list(range(n - recent, n)))
            out[t, h, :len(pick)] = torch.tensor(pick)
    return out


def attend(q, c, table, requests, positions, scale, pages=None):
    """(out, spread, reach, size): the attention, sum_j p_j |v_j| per element, and
    per row the largest scale * sum |q| |k| and the largest |v| of a key it sees."""
    T, Hq, d = q.shape
    P, H = c.k_scale.shape
    rep = Hq // H
    q = q.cpu().double()
    out = torch.zeros(T, Hq, d, dtype=torch.float64)
    spread = torch.zeros_like(out)
    reach, size = (torch.zeros(T, Hq, 1, dtype=torch.float64) for _ in range(2))
    for t in range(T):
        r, pos = requests[t], positions[t]
        if r < 0 or r >= len(table) or pos < 0:
            continue
        for h in range(H):
            lps = (range(min(pos // c.ps + 1, len(table[r]))) if pages is None
                   else [int(p) for p in pages[t, h]])
            ks, vs = [], []
            for lp in lps:
                if lp < 0 or lp >= len(table[r]) or not 0 <= table[r][lp] < P:
                    continue
                n = min(max(pos + 1 - lp * c.ps, 0), c.ps)
                pg = table[r][lp]
                ks.append(c.k[pg, h, :n, :d] * c.k_scale[pg, h])
                vs.append(c.v[pg, h, :n, :d] * c.v_scale[pg, h])
            if not ks or sum(k.shape[0] for k in ks) == 0:
                continue
            k, v = torch.cat(ks), torch.cat(vs)
            g = slice(h * rep, (h + 1) * rep)
            s = q[t, g] @ k.T * scale
            p = torch.softmax(s, 1)
            out[t, g], spread[t, g] = p @ v, p @ v.abs()
            reach[t, g, 0] = (q[t, g].abs() @ k.abs().T).amax(1) * abs(scale)
            size[t, g, 0] = v.abs().max()
    return out, spread, reach, size


def attend_tolerance(out, spread, reach, size, dtype, keys, d):
    """How far a result may be from `out`, per element.

    The result is rounded to its type once: off by finfo.eps / 2 of its value, or,
    below the type's normal numbers (f16's reach to 2^-14), by half the step that
    they all have, tiny * eps.  A
    probability p is rounded to f16 (fp32 queries: to three bf16 terms, 24 bits):
    off by 2^-11 of its value (2^-24), and where that f16 is subnormal by half its
    step, 2^-25: 2^-30 of the largest p, which is kept 2^5 above 1.  The numerator
    sum p v has these errors times |v|, the denominator sum p >= 1 those of the
    same rounded p, and the quotient is at most spread / 1: twice 2^-11 spread, and
    twice keys * 2^-30 * the largest |v|.  Products are exact; a score is a sum of
    d terms in fp32, off by (d + 2) 2^-24 of its terms' magnitudes (2^-23 where a
    step truncates), which enters the exponential, the sum and the maximum: twice.
    The exponential is off by 2^-22; the sums over the keys by keys * 2^-23 each,
    the numerator's and the denominator's."""
    half, least_step = torch.finfo(dtype).eps / 2, torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    term, least = (2.0 ** -24, 0.0) if dtype == torch.float32 else (2 * 2.0 ** -11, 2.0 ** -29)
    rel = term + 2 * (d + 2) * 2.0 ** -23 * reach + 2.0 ** -21 + 2 * keys * 2.0 ** -23
    return half * out.abs() + (1 + half) * (rel * spread + least * keys * size) + least_step / 2 + 2.0 ** -120
