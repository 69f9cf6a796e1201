"""Attention over shared prefixes and page copies against plain 64-bit implementations, at the sizes and tables where
they can go wrong.

Tolerances.  P is rounded to the cache's type for P.V (half a step u = eps / 2 of each p), o once more; a score is an
fp32 dot of 128 exact products, off by at most 128 * 2^-24 of sum |q_i k_i| * scale <= 12 for these inputs (9e-5,
which moves p and the sum of p alike).  With A = softmax . |v| in 64 bits:
    |o - want| <= A (u + 3e-4) + u |want| + n 2^-25 max|v| (fp16 only: p below its normal range)
    |lse - want| <= 1e-4 + 2^-22 |want|."""
import math

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
    """Rows (prefix or -1, own tokens, query tokens) over prefixes of the given page counts, on shuffled pages.  Planned
    for long rows (max_pages_per_row, a long kv_indices), or the small batches here would go to the ordinary kernels."""

    def __init__(self, hq, hkv, prefix_pages, rows, dtype="bf16", seed=0, num_pages=None, first_page=0, stale=None):
        g = torch.Generator(device=DEV)
        g.manual_seed(seed)
        self.hq, self.hkv, self.prefix_pages, self.rows = hq, hkv, prefix_pages, rows
        own = [max(1, -(-n // PAGE)) if n or p < 0 or p >= len(prefix_pages) else 0 for p, n, _ in rows]
        own = [0 if (n == 0 and p == -2) else c for c, (p, n, _) in zip(own, rows)]
        total = sum(prefix_pages) + sum(own)
        num_pages = num_pages or total + 2
        perm = (torch.randperm(num_pages - first_page, generator=torch.Generator().manual_seed(seed)) + first_page).tolist()
        it = iter(perm)
        self.shared = [[next(it) for _ in range(n)] for n in prefix_pages]
        self.pages = [(list(self.shared[p]) if 0 <= p < len(prefix_pages) else []) + [next(it) for _ in range(c)]
                      for (p, _, _), c in zip(rows, own)]
        self.kv_len = [(len(self.shared[p]) * PAGE if 0 <= p < len(prefix_pages) else 0) + n for p, n, _ in rows]
        last = [n - (len(pg) - 1) * PAGE if pg else 0 for n, pg in zip(self.kv_len, self.pages)]
        self.cache = torch.empty(num_pages, 2, PAGE, hkv, D, dtype=DT[dtype], device=DEV).normal_(0, 1, generator=g)
        if stale is not None:  # what lies behind a row's end
            for pg, n in zip(self.pages, last):
                if pg and n < PAGE:
                    self.cache[pg[-1], :, n:] = stale
        self.q = torch.empty(sum(r[2] for r in rows), hq, D, dtype=DT[dtype], device=DEV).normal_(0, 1, generator=g)
        self.qo = indptr([r[2] for r in rows])
        self.t = dict(kv_indptr=i32(indptr([len(p) for p in self.pages])), kv_indices=i32([x for p in self.pages for x in p] + [-1] * 65),
                      last=i32(last), row_prefix=i32([p for p, _, _ in rows]), prefix_indptr=i32(indptr(prefix_pages)),
                      prefix_indices=i32([x for s in self.shared for x in s]))

    def decode(self, **kw):
        t = self.t
        lse = torch.full((len(self.rows), self.hq), 7.0, device=DEV)
        kw.setdefault("max_pages_per_row", 8192)
        kw.setdefault("lse", lse)
        o = K.paged_decode_prefix(kw.pop("q", self.q), self.cache, t["kv_indptr"], t["kv_indices"], t["last"],
                                  t["row_prefix"], t["prefix_indptr"], t["prefix_indices"], **kw)
        return o, kw["lse"]

    def prefill(self, **kw):
        t = self.t
        q = kw.pop("q", self.q)
        kw.setdefault("lse", torch.full((q.shape[0], self.hq), 7.0, device=DEV))
        o = K.paged_prefill_prefix(q, self.cache, i32(self.qo), t["kv_indptr"], t["kv_indices"], t["last"],
                                   t["row_prefix"], t["prefix_indptr"], t["prefix_indices"],
                                   max_qo_len=max(r[2] for r in self.rows), **kw)
        return o, kw["lse"]

    def want(self, q=None, scale=1 / math.sqrt(D), tables=None):
        """(o, lse, A, max|v|, n) in 64 bits, row by row over the row's own page list; bad page ids are dropped."""
        q = (self.q if q is None else q).double()
        os, ls, As, ns = [], [], [], []
        for b, (pages, n) in enumerate(zip(tables or self.pages, self.kv_len)):
            x = q[self.qo[b]:self.qo[b + 1]]
            qn = x.shape[0]
            good = [0 <= p < self.cache.shape[0] for p in pages]
            kv = self.cache[torch.tensor([p if ok else 0 for p, ok in zip(pages, good)], dtype=torch.long, device=DEV)]
            kv = kv.double().transpose(0, 1).reshape(2, len(pages) * PAGE, self.hkv, D)[:, :n].repeat_interleave(self.hq // self.hkv, 2)
            k, v = kv[0].transpose(0, 1).contiguous(), kv[1].transpose(0, 1).contiguous()  # [hq, n, D]
            ok = torch.tensor(good, dtype=torch.bool, device=DEV).repeat_interleave(PAGE)[:n]
            seen = torch.ones(qn, n, dtype=torch.bool, device=DEV).tril(n - qn) & ok
            v = torch.where(ok[:, None], v, torch.zeros_like(v))
            z = (x.transpose(0, 1)[:, :, None] * k[:, None]).sum(-1) * scale if n * qn < 4096 else \
                torch.matmul(x.transpose(0, 1).contiguous(), k.transpose(1, 2).contiguous()) * scale
            z = torch.where(seen, z, torch.full_like(z, -math.inf))
            m = z.amax(-1, keepdim=True) if n else torch.full((self.hq, qn, 1), -math.inf, dtype=torch.float64, device=DEV)
            e = torch.exp(z - torch.where(m == -math.inf, torch.zeros_like(m), m))
            l = e.sum(-1, keepdim=True)
            p = torch.where(l > 0, e / l.clamp_min(1e-300), torch.zeros_like(e))
            os.append(torch.matmul(p, v).transpose(0, 1))
            As.append(torch.matmul(p, v.abs()).transpose(0, 1))
            ls.append((torch.where(m == -math.inf, torch.zeros_like(m), m) + l.log())[..., 0].transpose(0, 1))
            ns.append(torch.full((qn, 1, 1), float(n) * (float(v.abs().max()) if n else 0.0), device=DEV, dtype=torch.float64))
        return torch.cat(os), torch.cat(ls), torch.cat(As), torch.cat(ns)

    def check(self, got, want):
        o, lse = got
        wo, wl, A, nv = want
        eps = torch.finfo(o.dtype).eps
        u = eps / 2
        tol = A * (u + 3e-4) + u * wo.abs() + (nv * 2.0 ** -25 if o.dtype == torch.float16 else 0.0) + 1e-30
        bad = ((o.double() - wo).abs() > tol) | ~torch.isfinite(o.double())
        assert not bad.any(), f"o off at {bad.nonzero()[:4].tolist()}: {(o.double() - wo).abs().max():.3e}"
        empty = wl == -math.inf
        assert torch.equal(lse == -math.inf, empty)
        dl = (lse.double() - wl)[~empty].abs()
        assert (dl <= 1e-4 + 2.0 ** -22 * wl[~empty].abs()).all(), f"lse off by {dl.max():.3e}"


# ------------------------------------------------------------------ decode
HEADS = [(8, 8), (4, 2), (12, 4), (32, 8), (10, 2), (12, 2), (28, 4), (32, 4), (7, 1)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_decode_head_layouts(hq, hkv, dtype):
    """Every group size; three prefixes (one of a single page, one used by nobody), rows without one, own parts
    from one token on, ending at every place of a page."""
    rows = [(p, n, 1) for p, n in [(0, 1), (0, 16), (1, 17), (-1, 33), (0, 64), (1, 65), (0, 200), (-1, 1), (0, 100), (1, 5)]]
    b = Batch(hq, hkv, [19, 1, 7], rows, dtype, seed=hq)
    b.check(b.decode(), b.want())


@pytest.mark.parametrize("pages", [1, 3, 4, 5, 31, 257])
@pytest.mark.parametrize("batch", [1, 2, 9, 40, 130])
def test_decode_prefix_lengths(batch, pages):
    """Tiles of up to 32, 64 and 128 pairs and several tiles; prefixes that end inside a step."""
    b = Batch(12, 2, [pages], [(0, 1 + 7 * i % 50, 1) for i in range(batch)], seed=batch)
    b.check(b.decode(), b.want())


def test_decode_row_without_pages_and_prefix_of_whole_row():
    """A row without pages gives o = 0, lse = -inf; a row that is its prefix and nothing more; a prefix that does not
    fit in the row (a table of fewer tokens than the prefix's) leaves the row to its own pages."""
    b = Batch(32, 8, [6, 40], [(0, 0, 1), (-2, 0, 1), (0, 3, 1), (0, 0, 1)], seed=3)
    b.check(b.decode(), b.want())
    b.t["row_prefix"] = i32([1, 1, 1, 0])  # prefix 1 is longer than these rows
    b.check(b.decode(), b.want())


@pytest.mark.parametrize("junk", [-1, -7, 2, 1 << 30, -(1 << 31)])
def test_decode_row_prefix_outside_the_prefixes(junk):
    b = Batch(12, 2, [9, 5], [(0, 20, 1), (1, 3, 1), (0, 1, 1)], seed=5)
    b.t["row_prefix"] = i32([0, junk, 0])
    b.check(b.decode(), b.want())


def test_decode_no_prefixes_at_all():
    b = Batch(28, 4, [], [(-1, n, 1) for n in (1, 500, 16, 4000)], seed=6)
    b.check(b.decode(), b.want())


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_decode_stale_values_behind_the_rows(value):
    b = Batch(12, 2, [5], [(0, n, 1) for n in (1, 7, 15, 16, 30, 63)] + [(-1, 5, 1)], seed=7, stale=value)
    b.check(b.decode(), b.want())


@pytest.mark.parametrize("bad", [-1, 10 ** 6, -(1 << 31), (1 << 31) - 1])
def test_decode_pages_outside_the_cache_are_dropped(bad):
    """In the prefix's list (dropped for all its rows) and in a row's own; the dropped pages' V must not matter."""
    b = Batch(32, 8, [12], [(0, 100, 1), (0, 5, 1), (-1, 40, 1)], seed=8)
    b.cache[0] = math.nan  # what a masked load reads instead
    keep = [[p if p else 1 for p in r] for r in b.pages]
    shared = [p if p else 1 for p in b.shared[0]]
    shared[3] = shared[11] = bad
    rows = [shared + keep[0][12:], shared + keep[1][12:], keep[2]]
    rows[0][14] = bad
    b.t["prefix_indices"] = i32(shared)
    b.t["kv_indices"] = i32([p for r in rows for p in r] + [-1] * 65)
    b.check(b.decode(), b.want(tables=rows))


@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.0])
def test_decode_scales(scale):
    b = Batch(12, 2, [9], [(0, 20, 1), (0, 3, 1), (-1, 50, 1)], seed=9)
    b.q *= 0.2
    b.check(b.decode(sm_scale=scale), b.want(scale=scale))


def test_decode_strided_q_and_out():
    """q as a slice of the qkv projection's output, out as a slice of a wider buffer, whose rest stays."""
    b = Batch(12, 2, [9], [(0, 20, 1), (0, 3, 1), (-1, 50, 1)], seed=10)
    wide = torch.randn(3, 16 * D, device=DEV).to(torch.bfloat16)
    q = wide[:, :12 * D].view(3, 12, D)
    buf = torch.full((3, 20, D), 5.0, dtype=torch.bfloat16, device=DEV)
    got = b.decode(q=q, out=buf[:, 4:16])
    b.check(got, b.want(q=q))
    assert (buf[:, :4] == 5).all() and (buf[:, 16:] == 5).all()


def test_decode_many_rows_and_prefixes():
    """1024 rows, 300 prefixes, more than one table pass per block; some prefixes with one row, some with none."""
    rows = [((i * 7) % 290 if i % 5 else -1, 1 + i % 40, 1) for i in range(1024)]
    b = Batch(4, 2, [1 + i % 6 for i in range(300)], rows, seed=11)
    b.check(b.decode(), b.want())


def test_decode_long_prefix_and_a_long_lone_row():
    """Runs of many steps: a 40 000-token prefix under 20 rows, a row of 30 000 tokens alone."""
    rows = [(0, 1 + 13 * i, 1) for i in range(20)] + [(-1, 30000, 1)]
    b = Batch(12, 2, [2500], rows, seed=12)
    b.check(b.decode(), b.want())


def test_decode_more_pages_than_planned():
    """Rows longer than the planned maximum, in the kernels of a shared batch and of a small one."""
    b = Batch(12, 2, [200], [(0, 700 - 9 * i, 1) for i in range(70)], seed=13)
    b.check(b.decode(max_pages_per_row=60), b.want())
    b.check(b.decode(max_pages_per_row=4), b.want())


@pytest.mark.parametrize("batch", [1, 2, 7, 30])
def test_small_batches_on_the_ordinary_kernels(batch):
    """Planned for what they hold: each row by itself, the same results."""
    b = Batch(32, 8, [9], [(0 if i % 3 < 2 else -1, 1 + 11 * i % 40, 1) for i in range(batch)], seed=batch)
    most = max(len(p) for p in b.pages)
    assert batch * 8 * most <= 8192
    b.check(b.decode(max_pages_per_row=most), b.want())
    assert K.prefix_attention_workspace_bytes(batch, 32, 8, most) >= K.decode_workspace_bytes(batch, 32, 8, most)


def test_small_prompts_on_the_ordinary_kernel():
    b = Batch(32, 8, [9], [(0, 17, 17), (0, 1, 1), (-1, 30, 5), (0, 20, 6)], seed=24)
    b.t["kv_indices"] = b.t["kv_indices"][:-65].clone()
    assert b.t["kv_indices"].numel() <= 64
    b.check(b.prefill(), b.want())
    out = torch.full((29, 33 * D + 2), 2.0, dtype=torch.bfloat16, device=DEV)  # rows that only the shared kernel takes
    o = torch.as_strided(out, (29, 32, D), (33 * D + 2, D, 1), 2)
    b.check(b.prefill(out=o), b.want())
    assert (out[:, :2] == 2).all() and (out[:, 2 + 32 * D:] == 2).all()


def test_decode_cache_offsets_past_32_bits():
    """Pages whose byte and element offsets need more than 32 bits (8 kv heads: 64 KiB pages, 9 GB of them)."""
    b = Batch(8, 8, [40], [(0, 20, 1), (0, 3, 1), (-1, 50, 1)], seed=14, num_pages=140000, first_page=131000)
    b.check(b.decode(), b.want())


# ------------------------------------------------------------------ prompts
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_prefill_head_layouts(hq, hkv, dtype):
    """Rows of one token to several tiles, with and without own tokens in the cache before them; a row without any."""
    rows = [(0, 3, 3), (0, 40, 1), (-1, 70, 70), (1, 90, 30), (1, 0, 0), (0, 129, 129), (-1, 10, 1), (1, 300, 45), (0, 64, 64)]
    b = Batch(hq, hkv, [19, 1], rows, dtype, seed=hq)
    b.check(b.prefill(), b.want())


@pytest.mark.parametrize("pages,batch,qn", [(1, 1, 1), (3, 2, 17), (33, 40, 5), (257, 9, 33), (64, 3, 400), (500, 1, 31)])
def test_prefill_lengths(pages, batch, qn):
    b = Batch(32, 8, [pages], [(0, qn + 5 * i % 20, qn) for i in range(batch)], seed=pages)
    b.check(b.prefill(), b.want())


def test_prefill_prefix_that_reaches_into_the_query_tokens_is_not_applied():
    """7 pages of prefix, 118 tokens in all, 10 of them query tokens: the prefix would hide the causal mask."""
    b = Batch(32, 8, [7], [(0, 6, 6), (0, 30, 12)], seed=15)
    b.qo = [0, 10, 22]
    b.rows = [(0, 6, 10), (0, 30, 12)]
    b.q = torch.randn(22, 32, D, device=DEV).to(torch.bfloat16)
    b.check(b.prefill(), b.want())


def test_prefill_leaves_tokens_behind_the_last_row():
    b = Batch(12, 2, [7], [(0, 6, 6), (0, 30, 12)], seed=16)
    q = torch.randn(25, 12, D, device=DEV).to(torch.bfloat16)
    out, lse = torch.full_like(q, 3.0), torch.full((25, 12), 4.0, device=DEV)
    b.prefill(q=q, out=out, lse=lse)
    b.check((out[:18], lse[:18]), b.want(q=q))
    assert (out[18:] == 3).all() and (lse[18:] == 4).all()


@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_prefill_stale_values_behind_the_rows(value):
    b = Batch(12, 2, [5], [(0, 1, 1), (0, 23, 20), (-1, 77, 70)], seed=17, stale=value)
    b.check(b.prefill(), b.want())


def test_prefill_of_single_tokens_is_decode():
    b = Batch(28, 4, [50, 3], [(0, 40, 1), (1, 3, 1), (-1, 90, 1)] * 5, seed=18)
    for x, y in zip(b.prefill(), b.decode()):
        assert torch.equal(x, y)


# ------------------------------------------------------------------ streams, graphs
def test_same_bits_every_time_and_on_any_stream():
    b = Batch(32, 8, [300, 20], [(i % 2, 1 + 37 * i % 300, 1) for i in range(33)], seed=19)
    first = b.decode()
    side = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(6):
        with torch.cuda.stream(side[i % 2]):
            got.append(b.decode())
    torch.cuda.synchronize()
    for g in got:
        assert torch.equal(g[0], first[0]) and torch.equal(g[1], first[1])


def test_captured_decode_follows_the_tables():
    """A captured call replayed with other tables in the same buffers: rows that change prefix, lose it, get longer."""
    b = Batch(12, 2, [30, 11], [(0, 20, 1), (1, 3, 1), (0, 50, 1), (-1, 60, 1)], seed=20)
    c = Batch(12, 2, [12, 29], [(1, 33, 1), (1, 7, 1), (-1, 80, 1), (0, 9, 1)], seed=21, num_pages=b.cache.shape[0] + 40)
    b.cache = torch.cat([b.cache, torch.zeros_like(c.cache[:40])])
    room = {k: torch.zeros(max(v.numel(), c.t[k].numel()), dtype=torch.int32, device=DEV) for k, v in b.t.items()}
    cache, q = b.cache.clone(), b.q.clone()

    def load(x):
        for k, v in x.t.items():
            room[k][:v.numel()].copy_(v)
        cache.copy_(x.cache)
        q.copy_(x.q)

    def call(out, lse):
        K.paged_decode_prefix(q, cache, room["kv_indptr"], room["kv_indices"], room["last"], room["row_prefix"],
                              room["prefix_indptr"], room["prefix_indices"], max_pages_per_row=8192, out=out, lse=lse,
                              workspace=ws)

    ws = torch.empty(K.prefix_attention_workspace_bytes(4, 12, 2, 8192), dtype=torch.uint8, device=DEV)
    out, lse = torch.zeros_like(q), torch.zeros(4, 12, device=DEV)
    load(b)
    call(out, lse)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.inference_mode(), torch.cuda.graph(g):
        call(out, lse)
    for x in (b, c, c, b):
        load(x)
        out.fill_(9.0)
        lse.fill_(9.0)
        g.replay()
        torch.cuda.synchronize()
        x.check((out, lse), x.want())
        torch.randn(64, 64, device=DEV).sum().item()
    del g


# ------------------------------------------------------------------ refusals
def test_wrapper_refusals():
    b = Batch(12, 2, [9], [(0, 20, 1), (0, 3, 1)], seed=22)
    t = b.t
    with pytest.raises(TypeError, match="row_prefix must be int32"):
        b.t = {**t, "row_prefix": t["row_prefix"].long()}
        b.decode()
    with pytest.raises(ValueError, match="row_prefix needs"):
        b.t = {**t, "row_prefix": t["row_prefix"][:1]}
        b.decode()
    with pytest.raises(ValueError, match="prefix_indices must be contiguous"):
        b.t = {**t, "prefix_indices": t["prefix_indices"].repeat(2)[::2]}
        b.decode()
    b.t = t
    with pytest.raises(ValueError, match="workspace too small"):
        b.decode(workspace=torch.empty(256, dtype=torch.uint8, device=DEV))
    with pytest.raises(ValueError, match="lse must be"):
        b.decode(lse=torch.empty(2, 11, device=DEV))
    with pytest.raises(TypeError, match="q dtype"):
        b.decode(q=b.q.half())


# ------------------------------------------------------------------ page copies
def _caches(layers, pages, hkv, dtype, seed=0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return [torch.empty(pages, 2, PAGE, hkv, D, dtype=dtype, device=DEV).normal_(0, 1, generator=g) for _ in range(layers)]


def _plain_copy(caches, src, dst, tokens):
    out = [c.clone() for c in caches]
    for c, o in zip(caches, out):
        for s, d, t in zip(src, dst, tokens):
            if 0 <= s < c.shape[0] and 0 <= d < c.shape[0]:
                o[d, :, :max(0, min(t, PAGE))] = c[s, :, :max(0, min(t, PAGE))]
    return out


@pytest.mark.parametrize("hkv", [1, 2, 3, 4, 8, 16])
@pytest.mark.parametrize("layers", [1, 5, 130])
def test_copy_pages(layers, hkv):
    """Partial pages of every count, one source for several entries; more caches than one launch takes."""
    caches = _caches(layers, 60, hkv, torch.bfloat16)
    src = [3, 3, 3, 9, 10, 11, 12, 13, 14, 15, 16, 17, 18, 19, 20, 21, 22]
    dst = [40 + i for i in range(17)]
    tokens = list(range(17))
    want = _plain_copy(caches, src, dst, tokens)
    K.copy_pages(caches, i32(src), i32(dst), tokens=i32(tokens))
    assert all(torch.equal(c, w) for c, w in zip(caches, want))


def test_copy_whole_pages_past_32_bits():
    caches = _caches(1, 140000, 8, torch.float16)
    src, dst = [139999, 5, 70000], [0, 139998, 135000]
    want = caches[0][src].clone()
    before = caches[0][1].clone()
    K.copy_pages(caches, i32(src), i32(dst))
    assert torch.equal(caches[0][dst], want) and torch.equal(caches[0][1], before)


def test_copy_bad_entries_copy_nothing():
    caches = _caches(2, 12, 2, torch.bfloat16)
    src, dst, tokens = [1, -1, 2, 12, 3, 4, 5], [7, 8, -1, 9, 1 << 30, 4, 10], [16, 16, 16, 16, 16, 16, -3]
    want = _plain_copy(caches, src, dst, tokens)
    K.copy_pages(caches, i32(src), i32(dst), tokens=i32(tokens))
    assert all(torch.equal(c, w) for c, w in zip(caches, want))
    K.copy_pages(caches, i32([]), i32([]))
    assert all(torch.equal(c, w) for c, w in zip(caches, want))


def test_copy_in_a_captured_graph():
    caches = _caches(4, 40, 4, torch.bfloat16)
    src, dst, tokens = i32([0, 1, 2]), i32([20, 21, 22]), i32([16, 5, 9])
    start = [c.clone() for c in caches]
    K.copy_pages(caches, src, dst, tokens=tokens)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.inference_mode(), torch.cuda.graph(g):
        K.copy_pages(caches, src, dst, tokens=tokens)
    for s, d, t in (([0, 1, 2], [20, 21, 22], [16, 5, 9]), ([4, 4, 7], [30, 31, 20], [1, 16, 0])):
        for c, b in zip(caches, start):
            c.copy_(b)
        src.copy_(i32(s)), dst.copy_(i32(d)), tokens.copy_(i32(t))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(c, w) for c, w in zip(caches, _plain_copy(start, s, d, t)))
        torch.randn(64, 64, device=DEV).sum().item()
    del g


def test_copy_refusals():
    caches = _caches(2, 12, 2, torch.bfloat16)
    with pytest.raises(ValueError, match="no caches"):
        K.copy_pages([], i32([1]), i32([2]))
    with pytest.raises(ValueError, match="src names 2 pages, dst 1"):
        K.copy_pages(caches, i32([1, 2]), i32([2]))
    with pytest.raises(ValueError, match="tokens 1"):
        K.copy_pages(caches, i32([1, 2]), i32([3, 4]), tokens=i32([1]))
    with pytest.raises(ValueError, match="share a shape"):
        K.copy_pages(caches + _caches(1, 13, 2, torch.bfloat16), i32([1]), i32([2]))
    with pytest.raises(TypeError, match="src must be int32"):
        K.copy_pages(caches, torch.tensor([1], device=DEV), i32([2]))


# ------------------------------------------------------------------ the operators together
def test_fork_then_prompt_then_decode():
    """A sequence of 150 tokens forks: nine full pages are shared, its tenth page (6 tokens) is copied for each
    branch, each branch appends a prompt of its own, and a decode step follows; against every branch attending a
    cache of its own in which the whole context was written."""
    hq, hkv, n0, L = 12, 2, 150, 3
    caches = _caches(L, 80, hkv, torch.bfloat16, seed=30)
    pages0, branches = list(range(10)), [5, 23, 17]
    own = [[20 + 5 * i + k for k in range(3)] for i in range(3)]
    K.copy_pages(caches, i32([9] * 3), i32([o[0] for o in own]), tokens=i32([n0 % PAGE] * 3))
    for step, new in (("prompt", branches), ("decode", [1, 1, 1])):
        lens = [n0 + b + (step == "decode") for b in branches]
        npg = [-(-n // PAGE) for n in lens]
        rows = [pages0[:9] + o[:c - 9] for o, c in zip(own, npg)]
        ap = i32(indptr(new))
        ip, ind, last = i32(indptr(npg)), i32([p for r in rows for p in r] + [-1] * 65), i32([(n - 1) % PAGE + 1 for n in lens])
        for cache in caches:
            k = torch.randn(sum(new), hkv, D, device=DEV).to(torch.bfloat16)
            v = torch.randn(sum(new), hkv, D, device=DEV).to(torch.bfloat16)
            K.append_kv(k, v, ap, cache, ind, ip, last)
            q = torch.randn(sum(new), hq, D, device=DEV).to(torch.bfloat16)
            px = (i32([0, 0, 0]), i32([0, 9]), i32(pages0[:9]))
            if step == "prompt":
                o = K.paged_prefill_prefix(q, cache, ap, ip, ind, last, *px, max_qo_len=max(new))
                ref = K.paged_prefill(q, cache, ap, ip, ind, last, max_qo_len=max(new))
            else:
                o = K.paged_decode_prefix(q, cache, ip, ind, last, *px, max_pages_per_row=4096)
                ref = K.paged_decode(q, cache, ip, ind, last, max_pages_per_row=max(npg))
            # both round P and o once in bf16 (u = 2^-8 of values up to 4)
            assert (o.float() - ref.float()).abs().max() <= 4 * 4 * 2 ** -8
    assert torch.equal(caches[0][own[0][0], :, :6], caches[0][9, :, :6])
