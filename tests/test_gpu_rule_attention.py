"""Attention under score rules (capped, leaning by distance, windows, documents, prefixes) against a plain 64-bit
implementation, at the sizes, tables and masks where it can go wrong.

Tolerances.  P is rounded to the cache's type for P.V, each p_k to p_k (1 + d_k) with |d_k| <= u = eps / 2.  Divided by the
sum of the p_k that is off by sum p_k |d_k v_k| <= u A, divided by the rounded ones' sum by sum p_k |d_k (v_k - want)| <=
u (A + |want|); o is rounded once more.  A score is an fp32
sum of 128 exact products, off by at most 128 * 2^-24 of D = max sum |q_i k_i| * scale; the cap adds 2^-21 of the cap, and
the four roundings on the way to the exponent (scale, cap or bias, log2 e, maximum) 2^-21 of X, the largest |score| + |bias|
among the keys that weigh anything.  e = 2^-17 D + 2^-21 (cap + X) moves every p, and the sum of p, by a factor of at most
1 + 2 e together; exp2 and the sum add 2^-20.  With A = softmax . |v| in 64 bits:
    |o - want| <= A (u + 2 e + 2^-20) + 2 u |want| + n 2^-25 max|v| (fp16 only: p below its normal range)
    |lse - want| <= e + 2^-20 + 2^-21 |want|."""
import math
import random

import pytest
import torch

from delta_amd import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
PAGE, D = 16, 128
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def indptr(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


class Batch:
    """Rows of (cached tokens in all, query tokens) on shuffled pages of a paged cache."""

    def __init__(self, hq, hkv, rows, dtype="bf16", seed=0, q_std=1.5, first_page=0, num_pages=None, stale=math.nan):
        g = torch.Generator(device=DEV)
        g.manual_seed(seed)
        self.hq, self.hkv, self.rows, self.dtype = hq, hkv, rows, DT[dtype]
        counts = [-(-n // PAGE) for n, _ in rows]
        num_pages = num_pages or sum(counts) + 2
        order = torch.randperm(num_pages - first_page, generator=torch.Generator().manual_seed(seed))[:sum(counts) + 1]
        order = (order + first_page).tolist()
        at = indptr(counts)
        self.pages = [order[a:b] for a, b in zip(at, at[1:])]
        self.cache = torch.empty(num_pages, 2, PAGE, hkv, D, dtype=self.dtype, device=DEV)
        if first_page:  # (a large cache: only what is used)
            for p in order:
                self.cache[p].normal_(0, 1, generator=g)
        else:
            self.cache.normal_(0, 1, generator=g)
        for pg, (n, _) in zip(self.pages, rows):  # what lies behind a row's end
            if n % PAGE:
                self.cache[pg[-1], :, n % PAGE:] = stale
        self.qo = indptr([q for _, q in rows])
        self.T = self.qo[-1]
        self.q = torch.empty(self.T, hq, D, dtype=self.dtype, device=DEV).normal_(0, q_std, generator=g)
        self.tables = (i32(at), i32([p for pg in self.pages for p in pg] + [-1]),
                       i32([(n - 1) % PAGE + 1 if n else 0 for n, _ in rows]))
        self.pos = [n - ql + i for n, ql in rows for i in range(ql)]

    def prefill(self, rule, **kw):
        kw.setdefault("lse", torch.full((self.q.shape[0], self.hq), 7.0, device=DEV))
        q = kw.pop("q", self.q)
        o = K.paged_prefill_rule(q, self.cache, i32(self.qo), *self.tables, rule,
                                 max_qo_len=kw.pop("max_qo_len", max(1, max(q for _, q in self.rows))), **kw)
        return o, kw["lse"]

    def decode(self, rule, **kw):
        kw.setdefault("lse", torch.full((self.T, self.hq), 7.0, device=DEV))
        o = K.paged_decode_rule(kw.pop("q", self.q), self.cache, *self.tables, rule,
                                max_pages_per_row=kw.pop("max_pages_per_row", max(1, max(len(p) for p in self.pages))), **kw)
        return o, kw["lse"]

    def want(self, rule, scale=1 / math.sqrt(D), q=None):
        """o, lse, A, e and the fp16 term, in 64 bits, row by row."""
        q = (self.q if q is None else q).double()
        begin = rule.kv_begin.tolist() if rule.kv_begin is not None else None
        end = rule.kv_end.tolist() if rule.kv_end is not None else None
        outs = []
        for b, ((n, qn), pages) in enumerate(zip(self.rows, self.pages)):
            if qn == 0:
                continue
            t = self.qo[b]
            good = [0 <= p < self.cache.shape[0] for p in pages]
            ids = torch.tensor([p if ok else 0 for p, ok in zip(pages, good)], dtype=torch.long, device=DEV)
            kv = self.cache[ids].double().transpose(0, 1).reshape(2, -1, self.hkv, D)[:, :n]
            kv = kv.repeat_interleave(self.hq // self.hkv, 2).permute(0, 2, 1, 3).contiguous()
            k, v = kv[0], kv[1]  # [hq, n, D]
            key = torch.arange(n, device=DEV)
            pos = torch.arange(n - qn, n, device=DEV)[:, None]
            lo = torch.zeros_like(pos)
            if rule.window:
                lo = torch.maximum(lo, pos - rule.window + 1)
            if begin:
                lo = torch.maximum(lo, torch.tensor(begin[t:t + qn], device=DEV)[:, None])
            hi = torch.tensor(end[t:t + qn], device=DEV)[:, None] if end else pos + 1
            seen = (key >= lo) & (key < hi)
            seen &= torch.tensor(good, dtype=torch.bool, device=DEV).repeat_interleave(PAGE)[:n]
            x = q[t:t + qn].transpose(0, 1).contiguous()  # [hq, qn, D]
            z = torch.matmul(x, k.transpose(1, 2).contiguous()) * scale
            Dm = torch.matmul(x.abs(), torch.where(k.isfinite(), k.abs(), torch.zeros_like(k)).transpose(1, 2).contiguous()).amax(-1, keepdim=True) * abs(scale) if n else 0.0
            mag = z.abs()
            if rule.softcap:
                z = rule.softcap * torch.tanh(z / rule.softcap)
                mag = z.abs()
            if rule.slopes is not None:
                bias = rule.slopes.double()[:, None, None] * (pos - key).abs()
                z, mag = z - bias, mag + bias.abs()
            z = torch.where(seen, z, torch.full_like(z, -math.inf))
            m = z.amax(-1, keepdim=True) if n else z.new_full((self.hq, qn, 1), -math.inf)
            m0 = torch.where(m == -math.inf, torch.zeros_like(m), m)
            p = torch.exp(z - m0)
            l = p.sum(-1, keepdim=True)
            p = torch.where(l == 0, torch.zeros_like(p), p / l)
            X = torch.where(p > 2.0 ** -40, mag, torch.zeros_like(mag)).amax(-1, keepdim=True) if n else z.new_zeros(self.hq, qn, 1)
            # what is left out has no part in the result, whatever it holds
            o = torch.zeros(self.hq, qn, D, dtype=torch.float64, device=DEV)
            A = o.clone()
            if bool(v.isfinite().all()):
                o, A = torch.matmul(p, v), torch.matmul(p, v.abs())
            else:
                for i in range(qn):
                    s = seen[i]
                    o[:, i] = (p[:, i, s, None] * v[:, s]).sum(1)
                    A[:, i] = (p[:, i, s, None] * v[:, s].abs()).sum(1)
            e = 2.0 ** -17 * Dm + 2.0 ** -21 * (rule.softcap + X)
            vmax = float(torch.where(v.isfinite(), v.abs(), torch.zeros_like(v)).max()) if n else 0.0
            outs.append([y.transpose(0, 1) for y in (o, (m0 + l.log())[..., 0], A, e.expand(self.hq, qn, 1),
                                                     torch.full((self.hq, qn, 1), n * vmax, dtype=torch.float64, device=DEV))])
        return [torch.cat(c) for c in zip(*outs)]

    def check(self, got, want):
        o, lse = got
        wo, wl, A, e, nv = want
        o, lse = o[:wo.shape[0]], lse[:wo.shape[0]]
        u = torch.finfo(o.dtype).eps / 2
        nan = wl.isnan()
        assert torch.equal(lse.isnan(), nan) and o[nan].isnan().all()
        fin = wo.isfinite()
        assert torch.equal(o.isfinite() & ~nan[..., None], fin & ~nan[..., None]), "finite where it should not be, or the reverse"
        tol = A * (u + 2 * e + 2.0 ** -20) + 2 * u * wo.abs() + (nv * 2.0 ** -25 if o.dtype == torch.float16 else 0.0) + 1e-30
        bad = fin & ((o.double() - wo).abs() > tol)
        assert not bad.any(), f"o off at {bad.nonzero()[:4].tolist()}: {(o.double() - wo)[bad].abs().max():.3e}"
        empty = wl == -math.inf
        assert torch.equal(lse == -math.inf, empty) and (o[empty] == 0).all()
        ok = ~empty & ~nan
        d = (lse.double() - wl).abs() - (e[..., 0] + 2.0 ** -20 + 2.0 ** -21 * wl.abs())
        assert (d[ok] <= 0).all(), f"lse off by {d[ok].max():.3e} over its tolerance"


def slopes(hq):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)], device=DEV)


def documents(rows, seed):
    """Each query token's first key of its own document (documents of 1 to 90 tokens)."""
    rng, out = random.Random(seed), []
    for n, qn in rows:
        starts = [0]
        while starts[-1] < n:
            starts.append(starts[-1] + rng.randint(1, 90))
        out += [max(s for s in starts if s <= at) for at in range(n - qn, n)]
    return i32(out)


def prefixes(rows, seed):
    rng, out = random.Random(seed), []
    for n, qn in rows:
        pre = rng.randint(0, n)
        out += [max(at + 1, pre) for at in range(n - qn, n)]
    return i32(out)


def rule_of(kind, hq, rows, seed=0):
    return {"none": lambda: K.ScoreRule(),
            "cap": lambda: K.ScoreRule(softcap=30.0),
            "slopes": lambda: K.ScoreRule(slopes=slopes(hq)),
            "window1": lambda: K.ScoreRule(window=1),
            "window16": lambda: K.ScoreRule(window=16, softcap=5.0),
            "window100": lambda: K.ScoreRule(window=100),
            "docs": lambda: K.ScoreRule(kv_begin=documents(rows, seed)),
            "prefix": lambda: K.ScoreRule(kv_end=prefixes(rows, seed)),
            "all": lambda: K.ScoreRule(softcap=20.0, slopes=slopes(hq), window=77, kv_begin=documents(rows, seed),
                                       kv_end=prefixes(rows, seed))}[kind]()


KINDS = ["none", "cap", "slopes", "window1", "window16", "window100", "docs", "prefix", "all"]
# a lone token, whole prompts around a step's and a tile's ends, chunks, decode rows, no new token, an empty row
ROWS = [(1, 1), (5, 5), (64, 64), (130, 65), (200, 33), (777, 1), (50, 0), (130, 130), (0, 0), (17, 16), (129, 2)]
SINGLE = [(1, 1), (2, 1), (16, 1), (17, 1), (64, 1), (65, 1), (777, 1), (1500, 1), (31, 1)]
HEADS = [(32, 8), (28, 4), (40, 8), (12, 2), (3, 3), (4, 2), (9, 3), (16, 2)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hq,hkv,dtype", [(h, k, "bf16" if i % 2 else "fp16") for i, (h, k) in enumerate(HEADS)])
def test_prompts(hq, hkv, dtype, kind):
    b = Batch(hq, hkv, ROWS, dtype, seed=1, q_std=4.0)
    rule = rule_of(kind, hq, ROWS)
    b.check(b.prefill(rule), b.want(rule))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hq,hkv,dtype", [(h, k, "fp16" if i % 2 else "bf16") for i, (h, k) in enumerate(HEADS)])
def test_single_tokens(hq, hkv, dtype, kind):
    b = Batch(hq, hkv, SINGLE, dtype, seed=2, q_std=4.0)
    rule = rule_of(kind, hq, SINGLE)
    b.check(b.decode(rule), b.want(rule))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("kind", ["cap", "slopes", "window100", "docs", "all"])
@pytest.mark.parametrize("batch", [40, 150])
def test_single_tokens_of_many_rows(batch, kind, dtype):
    """Launches without splits, in balanced order and not."""
    rng = random.Random(batch)
    rows = [(rng.randint(1, 900), 1) for _ in range(batch)]
    b = Batch(32, 8, rows, dtype, seed=3)
    rule = rule_of(kind, 32, rows)
    b.check(b.decode(rule), b.want(rule))
    b.check(b.decode(rule, max_pages_per_row=700), b.want(rule))  # planned for longer rows
    b.check(b.decode(rule, max_pages_per_row=2), b.want(rule))    # and for shorter ones


@pytest.mark.parametrize("kind", ["cap", "slopes", "window100", "docs", "prefix", "all"])
@pytest.mark.parametrize("rows", [[(20000, 3)], [(9000, 40), (7000, 1), (5, 5)], [(6000, 1)] * 5 + [(200, 200)] * 3,
                                  [(4000, 17), (0, 0), (3, 0), (2500, 130)]])
def test_cut_rows(rows, kind):
    """Few tokens over long caches: parts of a row and their join, beside rows that are not cut."""
    b = Batch(28, 4, rows, "bf16", seed=4)
    rule = rule_of(kind, 28, rows)
    assert K.prefill_rule_workspace_bytes(b.T, len(rows), 28, 4, max(q for _, q in rows), b.tables[1].numel()) > 0
    want = b.want(rule)
    first = b.prefill(rule)
    b.check(first, want)
    again = b.prefill(rule, max_qo_len=700)  # planned for longer prompts
    b.check(again, want)
    rest = b.prefill(rule)
    assert torch.equal(first[0], rest[0]) and torch.equal(first[1], rest[1])


@pytest.mark.parametrize("hq,hkv", [(32, 8), (12, 2), (5, 5)])
@pytest.mark.parametrize("rows", [[(831, 1)], [(832, 1)], [(833, 3)], [(896, 40)], [(1535, 2)] * 6, [(1537, 9)] * 9,
                                  [(1100, 20)] * 24, [(1600, 4)] + [(100, 4)] * 30, [(3000, 1)] + [(40, 3)] * 70,
                                  [(30, 2)] * 64 + [(2500, 30), (0, 0), (70, 70), (4000, 1)]])
def test_around_the_least_cuts(rows, hq, hkv):
    """Row lengths and batches where the rows begin to be cut, batches that take more than one pass over the rows."""
    b = Batch(hq, hkv, rows, "bf16", seed=21)
    for rule in (K.ScoreRule(softcap=30.0), K.ScoreRule(window=1024, slopes=slopes(hq))):
        b.check(b.prefill(rule), b.want(rule))


# calls of 128 to 450 blocks: whole prompts, chunks, a long row that is cut beside short ones, rows of one step and none
FEW_HUNDRED = [[(700, 700)], [(400, 30)] * 30, [(1500, 40)] * 10 + [(6000, 1), (3000, 20)], [(0, 0), (1, 1), (63, 63), (64, 64)] * 12,
               [(129, 65), (190, 33), (65, 1)] * 8]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", FEW_HUNDRED)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_calls_of_a_few_hundred_blocks(rows, kind, dtype):
    b = Batch(32, 8, rows, dtype, seed=22, q_std=3.0)
    rule = rule_of(kind, 32, rows)
    b.check(b.prefill(rule), b.want(rule))


@pytest.mark.parametrize("what", [math.nan, math.inf])
@pytest.mark.parametrize("rows", [[(700, 700)], [(1500, 40)] * 10 + [(6000, 8), (3000, 20)]])
def test_a_few_hundred_blocks_beside_anything(rows, what):
    """Values that windows and documents leave out, and pages outside the cache."""
    b = Batch(32, 8, rows, seed=23)
    rng = random.Random(23)
    for pages in b.pages:
        for at in rng.sample(range(len(pages)), len(pages) // 4):
            b.cache[pages[at], 1, rng.randrange(PAGE), :, rng.randrange(D)] = what
    seen = K.ScoreRule(window=30, softcap=20.0)
    got, want = b.prefill(seen), b.want(seen)
    assert torch.equal(got[0].isfinite(), want[0].isfinite())
    assert torch.equal(got[1].isfinite(), want[1].isfinite())
    b = Batch(32, 8, rows, seed=24)
    for pages in b.pages:
        for at in rng.sample(range(len(pages)), len(pages) // 5):
            b.tables[1][sum(len(x) for x in b.pages[:b.pages.index(pages)]) + at] = pages[at] = rng.choice([-1, 1 << 30])
    for rule in (K.ScoreRule(), K.ScoreRule(softcap=30.0, slopes=slopes(32))):
        b.check(b.prefill(rule), b.want(rule))


@pytest.mark.parametrize("kind", ["cap", "slopes", "docs", "prefix"])
def test_long_prompts_in_wide_blocks(kind):
    rows = [(3600, 3600)]
    b = Batch(32, 8, rows, "bf16", seed=5, q_std=3.0)
    rule = rule_of(kind, 32, rows)
    b.check(b.prefill(rule), b.want(rule))


def test_more_query_tokens_than_cached_ones():
    """Positions in front of the cache see nothing; rows without a page, and tables without any."""
    rows = [(3, 10), (40, 5), (0, 4), (200, 230)]
    b = Batch(12, 2, rows, seed=17)
    for rule in (K.ScoreRule(), K.ScoreRule(softcap=9.0, window=2 ** 31 - 1), K.ScoreRule(window=5, slopes=slopes(12))):
        b.check(b.prefill(rule), b.want(rule))
    for call, rows in (("prefill", [(0, 3), (0, 1)]), ("decode", [(0, 1), (0, 1)])):
        b = Batch(12, 2, rows, seed=17)
        b.tables = (b.tables[0], i32([]), b.tables[2])
        o, lse = getattr(b, call)(K.ScoreRule(softcap=9.0))
        assert not o.any() and (lse == -math.inf).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("kind", ["none", "cap", "slopes", "all"])
def test_one_key_gives_its_value(kind, dtype):
    """A token that sees one key: its weight is 1 whatever its score, so o is that key's v to the bit."""
    rows = [(300, 300), (2500, 7), (40, 1)]
    b = Batch(12, 2, rows, dtype, seed=19, q_std=3.0)
    r = rule_of(kind, 12, rows)
    rng = random.Random(19)
    key = [rng.randint(0, p) for p in b.pos]
    rule = K.ScoreRule(softcap=r.softcap, slopes=r.slopes, kv_begin=i32(key), kv_end=i32([k + 1 for k in key]))
    row = [i for i, (_, n) in enumerate(rows) for _ in range(n)]
    page = torch.tensor([b.pages[i][k // PAGE] for i, k in zip(row, key)], device=DEV)
    v = b.cache[page, 1, torch.tensor(key, device=DEV) % PAGE].repeat_interleave(6, 1)
    assert torch.equal(b.prefill(rule)[0], v)
    assert torch.equal(b.prefill(rule, lse=None)[0], v)


@pytest.mark.parametrize("kind", KINDS)
def test_without_the_lse(kind):
    for rows in (ROWS, [(9000, 40), (7000, 1)]):
        b = Batch(28, 4, rows, "bf16", seed=20)
        rule = rule_of(kind, 28, rows)
        o, lse = b.prefill(rule)
        assert torch.equal(o, b.prefill(rule, lse=None)[0])


@pytest.mark.parametrize("tokens", [65, 80, 81, 300, 512, 513])
@pytest.mark.parametrize("hq,hkv,batch", [(12, 2, 3), (40, 8, 30), (16, 2, 1)])
def test_single_tokens_of_short_rows(hq, hkv, batch, tokens):
    rows = [(max(1, tokens - 37 * i), 1) for i in range(batch)]
    b = Batch(hq, hkv, rows, seed=18)
    rule = K.ScoreRule(softcap=30.0, slopes=slopes(hq), window=tokens - 3)
    b.check(b.decode(rule), b.want(rule))


def test_masks_that_leave_nothing():
    rows = [(40, 40), (100, 5), (3000, 4)]
    b = Batch(12, 2, rows, seed=6)
    begin = [p + 1 if i % 3 == 0 else 0 for i, p in enumerate(b.pos)]
    for rule in (K.ScoreRule(kv_begin=i32(begin)), K.ScoreRule(kv_end=i32([0] * b.T)), K.ScoreRule(kv_end=i32([-5] * b.T)),
                 K.ScoreRule(kv_begin=i32([1 << 30] * b.T), softcap=3.0), K.ScoreRule(kv_begin=i32([2 ** 31 - 1] * b.T), window=2),
                 K.ScoreRule(kv_begin=i32([-2 ** 31] * b.T), window=2 ** 31 - 1, kv_end=i32([2 ** 31 - 1] * b.T))):
        b.check(b.prefill(rule), b.want(rule))
    one = Batch(12, 2, [(40, 1), (3000, 1), (16, 1)], seed=6)
    for begin in ([40, 0, 15], [0, 3000, 16], [2 ** 31 - 1] * 3, [-2 ** 31] * 3):
        rule = K.ScoreRule(kv_begin=i32(begin))
        one.check(one.decode(rule), one.want(rule))
    rule = K.ScoreRule(kv_end=i32([0, 17, -1]))
    one.check(one.decode(rule), one.want(rule))


@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("rows", [[(300, 300), (70, 5)], [(5000, 20), (90, 90)]])
def test_what_masks_leave_out_may_hold_anything(rows, what):
    """Infinities and NaN in another document's keys and values, behind a window and behind the causal line."""
    for where in (0, 1):
        b = Batch(8, 2, rows, seed=7)
        n = rows[0][0]
        spoiled = [n - 20, n - 11, n // 2, 3]
        for s in spoiled:
            b.cache[b.pages[0][s // PAGE], where, s % PAGE, :, 5] = what
        begin = [(n - 10 if p >= n - 10 else n - 15 if p >= n - 15 else 0) if i < rows[0][1] else 0 for i, p in enumerate(b.pos)]
        for rule in (K.ScoreRule(), K.ScoreRule(window=8, softcap=30.0), K.ScoreRule(kv_begin=i32(begin), slopes=slopes(8))):
            got, want = b.prefill(rule), b.want(rule)
            if where == 1:
                b.check(got, want)
                continue
            # a key of infinity or NaN spoils the rows that see it: the others stay as they are
            sees = torch.zeros(b.T, dtype=torch.bool)
            for i, p in enumerate(b.pos[:rows[0][1]]):
                lo = max(0, p - rule.window + 1 if rule.window else 0, begin[i] if rule.kv_begin is not None else 0)
                sees[i] = any(lo <= s <= p for s in spoiled)
            keep = ~sees.to(DEV)
            assert got[0][keep].isfinite().all()
            part = [w[keep] for w in want]
            b.check((got[0][keep], got[1][keep]), part)


@pytest.mark.parametrize("what", [math.nan, math.inf])
def test_single_token_beside_anything(what):
    b = Batch(8, 2, [(300, 1), (40, 1)], seed=8, stale=what)
    for s in (0, 250, 287):
        b.cache[b.pages[0][s // PAGE], :, s % PAGE] = what
    rule = K.ScoreRule(window=12)
    b.check(b.decode(rule), b.want(rule))
    rule = K.ScoreRule(kv_begin=i32([288, 3]), softcap=9.0)
    b.check(b.decode(rule), b.want(rule))
    got = b.decode(K.ScoreRule())  # sees them
    assert got[0][0].isnan().any() and got[0][1].isfinite().all()


@pytest.mark.parametrize("single", [False, True])
def test_pages_outside_the_cache_are_dropped(single):
    rows = [(200, 1), (90, 1), (2000, 1)] if single else [(200, 50), (90, 90), (2000, 7)]
    b = Batch(12, 2, rows, seed=9)
    ids, at = b.tables[1], 0
    for r, j, bad in ((0, 2, -1), (0, 12, 1 << 30), (1, 0, b.cache.shape[0]), (2, 100, -7)):
        b.pages[r][j] = bad
        ids[sum(len(p) for p in b.pages[:r]) + j] = bad
    for rule in (K.ScoreRule(softcap=30.0), K.ScoreRule(window=60, slopes=slopes(12))):
        b.check(b.decode(rule) if single else b.prefill(rule), b.want(rule))


@pytest.mark.parametrize("padded", [30, 2900, 2992, 3008, 3009, 9000])
def test_few_tokens_of_many_planned(padded):
    """A query buffer planned for more tokens than the rows have, up to more than the pages hold."""
    b = Batch(12, 2, [(2990, 7), (9, 2)], seed=25)
    q = torch.zeros(padded, 12, D, dtype=b.dtype, device=DEV)
    q[:9] = b.q
    rule = K.ScoreRule(softcap=30.0)
    for most in (7, padded):
        o, lse = torch.full_like(q, 5.0), torch.full((padded, 12), 5.0, device=DEV)
        b.check(b.prefill(rule, q=q, out=o, lse=lse, max_qo_len=most), b.want(rule))
        assert (o[9:] == 5.0).all() and (lse[9:] == 5.0).all()


def test_tokens_behind_the_last_row_stay():
    b = Batch(12, 2, [(40, 40), (900, 3)], seed=10)
    q = torch.cat([b.q, torch.full((9, 12, D), math.nan, dtype=b.dtype, device=DEV)])
    o = torch.full_like(q, 3.0)
    lse = torch.full((q.shape[0], 12), 5.0, device=DEV)
    rule = K.ScoreRule(softcap=30.0)
    got = b.prefill(rule, q=q, out=o, lse=lse)
    b.check(got, b.want(rule, q=q))
    assert (o[b.T:] == 3.0).all() and (lse[b.T:] == 5.0).all()


@pytest.mark.parametrize("single", [False, True])
def test_strides(single):
    """q and out as views of wider rows, heads apart."""
    rows = [(200, 1), (90, 1)] if single else [(200, 50), (90, 90)]
    b = Batch(8, 2, rows, "fp16", seed=11)
    wide = torch.randn(b.T, 24, 136, device=DEV).to(b.dtype)
    wide[:, 3:19:2, :D] = b.q
    out = torch.full((b.T, 24, 132), 9.0, dtype=b.dtype, device=DEV)
    rule = K.ScoreRule(softcap=30.0, slopes=slopes(8))
    call = b.decode if single else b.prefill
    view = out[:, 2:18:2, :D]
    got = call(rule, q=wide[:, 3:19:2, :D], out=view)
    assert got[0].data_ptr() == view.data_ptr()
    b.check(got, b.want(rule))
    assert (out[:, 1::2] == 9.0).all() and (out[..., D:] == 9.0).all()
    plain = call(rule)
    assert torch.equal(plain[0], got[0])


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1.0])
def test_scales(scale):
    rows = [(150, 40), (70, 70)]
    b = Batch(8, 2, rows, seed=12, q_std=0.5)
    for rule in (K.ScoreRule(), K.ScoreRule(softcap=4.0), K.ScoreRule(slopes=slopes(8)), K.ScoreRule(window=9)):
        b.check(b.prefill(rule, sm_scale=scale), b.want(rule, scale))
    one = Batch(8, 2, [(150, 1), (7, 1)], seed=12, q_std=0.5)
    for rule in (K.ScoreRule(softcap=4.0), K.ScoreRule(slopes=slopes(8))):
        one.check(one.decode(rule, sm_scale=scale), one.want(rule, scale))


@pytest.mark.parametrize("cap", [1e-3, 0.5, 1e4, 1e20])
def test_caps_of_any_size(cap):
    rows = [(150, 40), (70, 70)]
    b = Batch(8, 2, rows, seed=13, q_std=4.0)
    rule = K.ScoreRule(softcap=cap)
    want = b.want(rule)
    if cap >= 1e4:  # far above the scores: no error that grows with the cap
        want[3] = want[3] - 2.0 ** -21 * cap
    b.check(b.prefill(rule), want)
    one = Batch(8, 2, [(150, 1), (7, 1)], seed=13, q_std=4.0)
    want = one.want(rule)
    if cap >= 1e4:
        want[3] = want[3] - 2.0 ** -21 * cap
    one.check(one.decode(rule), want)


def test_without_a_rule_it_is_the_causal_attention():
    rows = [(150, 40), (70, 70), (1000, 1)]
    b = Batch(32, 8, rows, seed=14)
    got = b.prefill(K.ScoreRule())
    lse = torch.empty_like(got[1])
    o = K.paged_prefill(b.q, b.cache, i32(b.qo), *b.tables, max_qo_len=70, lse=lse)
    b.check((o, lse), b.want(K.ScoreRule()))
    b.check(got, b.want(K.ScoreRule()))


@pytest.mark.parametrize("single", [False, True])
def test_cache_offsets_past_32_bits(single):
    """Pages past 2^31 elements (4 GiB) of the cache."""
    rows = [(700, 1), (90, 1)] if single else [(700, 30), (90, 90)]
    b = Batch(32, 8, rows, seed=15, first_page=66000, num_pages=66100)
    assert min(min(p) for p in b.pages) * 2 * PAGE * 8 * D > 2 ** 31
    rule = K.ScoreRule(softcap=30.0, window=500)
    b.check(b.decode(rule) if single else b.prefill(rule), b.want(rule))


@pytest.mark.parametrize("single", [False, True])
@torch.inference_mode()  # as the engine captures: torch's graph state must not change mode between captures
def test_graphs_and_streams(single):
    """Two captured calls that share a workspace, replayed with eager work between, and a call on a stream of its own."""
    rows = [(5000, 1), (300, 1)] if single else [(5000, 20), (300, 70)]
    b = Batch(28, 4, rows, seed=16)
    rules = [K.ScoreRule(softcap=30.0), K.ScoreRule(slopes=slopes(28), window=900)]
    call = b.decode if single else b.prefill
    want = [b.want(r) for r in rules]
    eager = [call(r) for r in rules]
    nbytes = K.decode_rule_workspace_bytes(2, 28, 4, 313) if single else \
        K.prefill_rule_workspace_bytes(b.T, 2, 28, 4, 70, b.tables[1].numel())
    assert nbytes > 0
    ws = torch.empty(nbytes, dtype=torch.uint8, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call(rules[0])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], eager[0][0]) and torch.equal(got[1], eager[0][1])
    outs, graphs = [], []
    for r in rules:
        o, lse = torch.empty_like(b.q), torch.empty(b.T, 28, device=DEV)
        qo = i32(b.qo)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            if single:
                K.paged_decode_rule(b.q, b.cache, *b.tables, r, max_pages_per_row=313, out=o, lse=lse, workspace=ws)
            else:
                K.paged_prefill_rule(b.q, b.cache, qo, *b.tables, r, max_qo_len=70, out=o, lse=lse, workspace=ws)
        graphs.append((g, qo))
        outs.append((o, lse))
    for _ in range(3):
        for (g, _), (o, lse), w, e in zip(graphs, outs, want, eager):
            o.fill_(5.0)
            lse.fill_(5.0)
            ws.fill_(255)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(lse, e[1]) and torch.equal(o, e[0])
            b.check((o, lse), w)
            b.check(call(rules[0]), want[0])


@pytest.mark.parametrize("seed", range(12))
def test_drawn(seed):
    rng = random.Random(seed)
    hq, hkv = rng.choice(HEADS)
    rows = []
    for _ in range(rng.choice([1, 2, 7, 70])):
        n = int(math.exp(rng.uniform(0, math.log(3000))))
        rows.append((n, rng.choice([0, 1, min(n, rng.randint(1, 40)), min(n, 300)])))
    if not sum(q for _, q in rows):
        rows.append((9, 4))
    b = Batch(hq, hkv, rows, rng.choice(["bf16", "fp16"]), seed=seed, q_std=rng.choice([1.0, 4.0]))
    rule = K.ScoreRule(softcap=rng.choice([0.0, 15.0, 50.0]), slopes=rng.choice([None, slopes(hq)]),
                       window=rng.choice([0, 0, rng.randint(1, 2000)]),
                       kv_begin=rng.choice([None, documents(rows, seed)]), kv_end=rng.choice([None, prefixes(rows, seed)]))
    b.check(b.prefill(rule), b.want(rule))


# (q heads, kv heads, rows, planned tokens): one set of waves to a block, two, eight waves to a block, cut rows
BLOCKS = [(8, 2, [(300, 40), (70, 70), (20, 31)], 70), (32, 8, [(700, 700), (9, 14)], 700), (32, 8, [(290, 200), (5, 9)], 4000),
          (28, 4, [(5000, 40), (90, 90)], 90)]


@pytest.mark.parametrize("what", [math.nan, math.inf])
@pytest.mark.parametrize("kind", ["none", "cap", "slopes", "all"])
@pytest.mark.parametrize("blocks", range(len(BLOCKS)))
def test_tokens_without_keys_beside_anything(blocks, kind, what):
    """Tokens that see no key (bounds, positions in front of the cache, pages outside it) among tokens whose values are NaN or
    infinity: 0 and -inf, as beside finite values."""
    hq, hkv, rows, most = BLOCKS[blocks]
    rng = random.Random(blocks)
    for dtype in ("bf16", "fp16"):
        b = Batch(hq, hkv, rows, dtype, seed=30, q_std=3.0)
        r = rule_of(kind if kind != "all" else "cap", hq, rows)
        n = rows[0][0]
        for s in range(n % 7, n, 9):
            b.cache[b.pages[0][s // PAGE], 1, s % PAGE, :, rng.randrange(D)] = what
        b.cache[b.pages[-1][0], 1, 1] = what
        bad = n // PAGE - 1  # a page outside the cache, and tokens that see nothing else
        b.pages[0][bad] = b.tables[1][bad] = -1
        begin = [p + 1 if i % 3 == 0 else PAGE * bad if i % 3 == 1 else 0 for i, p in enumerate(b.pos)]
        end = [0 if i % 4 == 0 else PAGE * bad + PAGE if i % 3 == 1 else p + 1 for i, p in enumerate(b.pos)]
        for kb, ke in ((begin, None), (begin, end), (None, end), (None, None)):
            rule = K.ScoreRule(softcap=r.softcap, slopes=slopes(hq) if kind in ("slopes", "all") else None,
                               kv_begin=kb and i32(kb), kv_end=ke and i32(ke))
            b.check(b.prefill(rule, max_qo_len=most), b.want(rule))


def far_cap(want, cap):
    """A cap far above the scores: no error that grows with it."""
    want[3] = want[3] - 2.0 ** -21 * cap
    return want


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("cap", [1e3, 1e4, 1e20])
@pytest.mark.parametrize("size", [math.inf, -math.inf, "max"])
@pytest.mark.parametrize("single", [False, True])
def test_large_caps_beside_hidden_keys_of_any_size(single, size, cap, dtype):
    """Keys behind a row's end, in front of its first one and in place of a page outside the cache have no part in how the
    scores of the others are capped."""
    rows = [(300, 1), (41, 1), (200, 1)] if single else [(300, 40), (41, 41), (200, 5)]
    b = Batch(8, 2, rows, dtype, seed=31, q_std=3.0, stale=0.0, first_page=1, num_pages=40)
    b.cache[0] = 0.0
    call, size = b.decode if single else b.prefill, torch.finfo(DT[dtype]).max if size == "max" else size
    b.tables[1][sum(len(p) for p in b.pages[:2]) + 4] = b.pages[2][4] = -1
    begin = i32([251 if i < rows[0][1] else 0 for i in range(b.T)])
    rules = [K.ScoreRule(softcap=cap, kv_begin=begin), K.ScoreRule(softcap=cap, kv_begin=begin, slopes=slopes(8))]
    want = [far_cap(b.want(rule), cap) for rule in rules]  # (of the values that are seen)
    b.cache[b.pages[0][-1], 0, 300 % PAGE:, :, 5] = size
    b.cache[b.pages[1][-1], 0, 41 % PAGE:, :, 5] = size
    b.cache[b.pages[0][250 // PAGE], 0, 250 % PAGE, :, 7] = size
    b.cache[0, 0, :, :, 9] = size
    for rule, w in zip(rules, want):
        b.check(call(rule), w)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("cap", [1e3, 1e6])
@pytest.mark.parametrize("single", [False, True])
def test_large_caps_beside_tokens_and_heads_of_larger_scores(single, cap, dtype):
    """Scores about the cap in some tokens and heads; the small ones beside them keep an error of their own size."""
    rows = [(300, 1), (41, 1)] if single else [(300, 40), (41, 41)]
    b = Batch(8, 2, rows, dtype, seed=32, q_std=3.0)
    b.q[::3, ::4] *= cap / 20
    rule = K.ScoreRule(softcap=cap)
    call = b.decode if single else b.prefill
    b.check(call(rule), far_cap(b.want(rule), cap))


def saturate(b, sign, cap, scale):
    """Scores of about sign * cap throughout, values of about `scale`."""
    g = torch.Generator(device=DEV)
    g.manual_seed(33)
    u = torch.empty(b.hkv, D, device=DEV).normal_(0, 1, generator=g).sign()
    b.cache[:, 0] = (u + 0.3 * b.cache[:, 0].float()).to(b.dtype)
    b.cache[:, 1] *= scale
    far = torch.linspace(0.1, 0.35, b.T, device=DEV)[:, None, None] * cap  # raw scores from 1.1 to 4 caps
    b.q = (sign * far * u.repeat_interleave(b.hq // b.hkv, 0) + 0.3 * b.q.float()).to(b.dtype)


@pytest.mark.parametrize("power", [-40, -20, -10, 0, 20, 40, 60, 100])
@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("cap", [30.0, 45.0, 50.0, 54.0, 55.0, 64.0, 65.0])
def test_scores_at_the_cap(cap, sign, power):
    """Rows whose every score is about -cap or cap, where p is smallest and largest beside a constant reference, with values from
    small to large: one set of waves, two, eight waves, cut rows, tokens of one key."""
    dtypes = ["bf16", "fp16"] if -10 <= power <= 0 else ["bf16"]
    for dtype in dtypes:
        for hq, hkv, rows, most in BLOCKS:
            b = Batch(hq, hkv, [(n, min(n, q)) for n, q in rows], dtype, seed=34, stale=0.0)
            saturate(b, sign, cap, 2.0 ** power)
            rule = K.ScoreRule(softcap=cap)
            b.check(b.prefill(rule, max_qo_len=most), b.want(rule))
        key = [p * 5 // 7 for p in b.pos]
        rule = K.ScoreRule(softcap=cap, kv_begin=i32(key), kv_end=i32([k + 1 for k in key]))
        row = [i for i, (_, n) in enumerate(b.rows) for _ in range(n)]
        page = torch.tensor([b.pages[i][k // PAGE] for i, k in zip(row, key)], device=DEV)
        v = b.cache[page, 1, torch.tensor(key, device=DEV) % PAGE].repeat_interleave(hq // hkv, 1)
        assert torch.equal(b.prefill(rule)[0], v)


@pytest.mark.parametrize("sign", [-1, 1])
def test_parts_of_a_row_at_both_ends_of_the_cap(sign):
    """A cut row of which some keys score -64 and others, in other parts, anything: the parts' sums have references of their own."""
    for power in (-30, 0, 60):
        b = Batch(28, 4, [(6000, 12), (3000, 5)], seed=35, stale=0.0)
        saturate(b, -1, 64.0, 2.0 ** power)
        pages = torch.tensor(b.pages[0][40:90], device=DEV)  # 800 keys
        b.cache[pages, 0] *= -0.02 if sign < 0 else -1.0
        rule = K.ScoreRule(softcap=64.0)
        b.check(b.prefill(rule), b.want(rule))


def test_rows_cut_in_a_call_of_very_many_steps():
    """A row of 400000 pages cut in three beside prompts of 2^24 tile steps and more, the same pages over and over: as the row
    alone, which is cut in some hundred.

    A part adds up to 34000 sums of 64 keys, each addition off by 2^-24 of the sum: 2^-8.9 of l, le and every element's A at most,
    beside what the file's head counts (scores to 2^-16: D < 16, cap 30)."""
    pages = 32768
    g = torch.Generator(device=DEV)
    g.manual_seed(36)
    cache = torch.empty(pages, 2, PAGE, 1, D, dtype=torch.bfloat16, device=DEV).normal_(0, 1, generator=g)
    cache[:, 1] += 1.0
    rows = [(400000, 5)] + [(pages, 700)] * 48 + [(1, 1)]
    kv = indptr([n for n, _ in rows])
    table = torch.arange(kv[-1], dtype=torch.int32, device=DEV) % pages
    qo = indptr([n for _, n in rows])
    q = torch.empty(qo[-1], 8, D, dtype=torch.bfloat16, device=DEV).normal_(0, 1, generator=g)
    rule = K.ScoreRule(softcap=30.0)

    def call(r0, r1):
        t = slice(qo[r0], qo[r1])
        most, n = max(n for _, n in rows[r0:r1]), q[t].shape[0]
        lse = torch.empty(n, 8, device=DEV)
        ids = table[kv[r0]:kv[r1]]
        need = K.prefill_rule_workspace_bytes(n, r1 - r0, 8, 1, most, ids.numel())
        ws = torch.full((need,), 255, dtype=torch.uint8, device=DEV)  # (NaN)
        o = K.paged_prefill_rule(q[t], cache, i32([x - qo[r0] for x in qo[r0:r1 + 1]]), i32([x - kv[r0] for x in kv[r0:r1 + 1]]), ids,
                                 i32([PAGE] * (r1 - r0)), rule, max_qo_len=most, lse=lse, workspace=ws)
        return o.double(), lse.double(), need

    o, lse, need = call(0, len(rows))
    assert need > 0
    for r in (0, 7, 49):
        alone, lone, _ = call(r, r + 1)
        t = slice(qo[r], qo[r + 1])
        A, off = alone.abs().max() + 3.0, 2.0 ** -8.9  # (E|v - 1| < 1; one key's |v| is below its own |o| + 3)
        assert (o[t] - alone).abs().max() <= 2 * (A * (2.0 ** -8 + 2.0 ** -15 + 2 * off) + 2.0 ** -7 * A)
        assert (lse[t] - lone).abs().max() <= 2 * (2.0 ** -13 + off + 2.0 ** -21 * 60)


@pytest.mark.parametrize("hq,hkv", [(32, 32), (40, 40), (68, 17)])
def test_single_tokens_of_many_kv_heads(hq, hkv):
    """More kv heads than the decode call takes: refused there, a prompt call of one token a row."""
    b = Batch(hq, hkv, SINGLE, seed=37, q_std=3.0)
    rule = K.ScoreRule(slopes=slopes(hq), window=700)
    with pytest.raises(RuntimeError, match="num_kv_heads .* > 16 unsupported"):
        b.decode(rule)
    b.check(b.prefill(rule, max_qo_len=1), b.want(rule))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("kind", ["none", "cap", "slopes", "window", "docs"])
@pytest.mark.parametrize("rows", [[(700, 700)], [(1500, 40)] * 10 + [(6000, 8), (3000, 20)]])
def test_values_beside_anything_in_a_few_hundred_blocks(rows, kind, what, dtype):
    """Two sets of waves to a block: rows that are summed again, because of values that they do not see, against 64 bits."""
    b = Batch(32, 8, rows, dtype, seed=38, q_std=3.0)
    rng = random.Random(38)
    for pages, (n, qn) in zip(b.pages, rows):
        for s in rng.sample(range(n - qn // 2 - 8, n - 1), 5) + [n // 3]:
            b.cache[pages[s // PAGE], 1, s % PAGE, :, rng.randrange(D)] = what
    rule = {"none": K.ScoreRule(), "cap": K.ScoreRule(softcap=30.0), "slopes": K.ScoreRule(slopes=slopes(32)),
            "window": K.ScoreRule(window=30, softcap=20.0), "docs": K.ScoreRule(kv_begin=documents(rows, 38))}[kind]
    got, want = b.prefill(rule), b.want(rule)
    assert 0.5 < want[0].isfinite().double().mean() < 1
    b.check(got, want)


@pytest.mark.parametrize("kind", KINDS)
def test_single_tokens_by_either_call(kind):
    for hq, hkv, dtype in ((12, 2, "bf16"), (40, 8, "fp16")):
        b = Batch(hq, hkv, SINGLE, dtype, seed=39, q_std=4.0)
        rule = rule_of(kind, hq, SINGLE)
        want = b.want(rule)
        b.check(b.prefill(rule), want)
        b.check(b.decode(rule), want)
