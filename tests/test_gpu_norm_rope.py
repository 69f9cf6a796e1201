"""Norms and rotation of queries and keys, with and without the append, against a plain 64-bit implementation.

Tolerances.  The result is rounded once (u = eps / 2 of it; fp16 below its normal range half of 2^-24).  Before that, in
fp32: the sum of 128 squares takes 12 roundings deep, the root, the reciprocal and the two factors five more (2^-24 each, so
2^-20 of a normalised element at most), an angle's (cos, sin) are off by 2^-22 at most (a turn's fraction of 2^-25, pi, the
function's own two steps), the two products and their sum by three roundings.  So, with a and b the pair's normalised
elements: |y - want| <= u |want| + factor (|a| + |b|) 2^-19 + (fp16) 2^-25."""
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


def turned(x, w, eps, freqs, factor, pos, interleaved):
    """(want, tolerance without the rounding) of [T, heads, 128] in 64 bits."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    y, slack = x.clone(), x.abs() * 2.0 ** -19
    P = len(freqs)
    angle = torch.tensor(pos, dtype=torch.float64, device=DEV)[:, None] * torch.tensor(freqs, dtype=torch.float64, device=DEV)
    c, s = torch.cos(angle)[:, None] * factor, torch.sin(angle)[:, None] * factor
    ia = torch.arange(P, device=DEV) * 2 if interleaved else torch.arange(P, device=DEV)
    ib = ia + 1 if interleaved else ia + P
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    slack[..., ia] = slack[..., ib] = abs(factor) * (a.abs() + b.abs()) * 2.0 ** -19
    return y, slack


def check(got, want, slack):
    u = torch.finfo(got.dtype).eps / 2
    tol = u * want.abs() + slack + (2.0 ** -25 if got.dtype == torch.float16 else 1e-38)
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), f"off at {bad.nonzero()[:4].tolist()}: {(got.double() - want)[bad].abs().max():.3e}"


class Step:
    """A prompt or decode step: rows of (cached tokens in all, new tokens), q, k and v views of a merged projection."""

    def __init__(self, hq, hkv, rows, dtype="bf16", seed=0, first=None, norm=True, pad=0, std=1.0):
        g = torch.Generator(device=DEV)
        g.manual_seed(seed)
        self.hq, self.hkv, self.rows = hq, hkv, rows
        self.T = sum(q for _, q in rows)
        qkv = torch.empty(self.T + pad, (hq + 2 * hkv) * D, dtype=DT[dtype], device=DEV).normal_(0, std, generator=g)
        q, k, v = qkv.split([hq * D, hkv * D, hkv * D], -1)
        self.q, self.k, self.v = q.unflatten(-1, (hq, D)), k.unflatten(-1, (hkv, D)), v.unflatten(-1, (hkv, D))
        self.first = first or [n - ql for n, ql in rows]
        self.pos = [f + i for f, (_, ql) in zip(self.first, rows) for i in range(ql)]
        self.ip, self.off = i32(indptr([ql for _, ql in rows])), i32(self.first)
        self.w = {"q_weight": None, "k_weight": None}
        if norm:
            self.w = {n: torch.empty(D, dtype=DT[dtype], device=DEV).normal_(1, 0.3, generator=g) for n in self.w}
        counts = [-(-n // PAGE) for n, _ in rows]
        order = torch.randperm(sum(counts) + 3, generator=torch.Generator().manual_seed(seed)).tolist()
        at = indptr(counts)
        self.pages = [order[a:b] for a, b in zip(at, at[1:])]
        self.cache = torch.empty(len(order), 2, PAGE, hkv, D, dtype=DT[dtype], device=DEV).normal_(0, 1, generator=g)
        self.tables = (i32([p for pg in self.pages for p in pg]), i32(at), i32([(n - 1) % PAGE + 1 if n else 0 for n, _ in rows]))

    def append(self, rot, cache=None, **kw):
        cache = self.cache.clone() if cache is None else cache
        return K.qk_norm_rope_append(self.q, self.k, self.v, self.ip, self.off, cache, *self.tables, rot, **self.w, **kw), cache

    def rope(self, rot, **kw):
        return K.qk_norm_rope(self.q, self.k, self.ip, self.off, rot, **self.w, **kw)

    def want(self, freqs, factor, interleaved, eps=1e-6):
        t = slice(0, self.T)
        return [turned(x[t], w, eps, freqs, factor, self.pos, interleaved)
                for x, w in ((self.q, self.w["q_weight"]), (self.k, self.w["k_weight"]))]

    def check_cache(self, cache, k_want, k_slack):
        """Every new token's slot, and everything else as it was."""
        after = self.cache.clone()
        t = 0
        for (n, ql), pg in zip(self.rows, self.pages):
            for i in range(ql):
                s = n - ql + i
                check(cache[pg[s // PAGE], 0, s % PAGE], k_want[t], k_slack[t])
                assert torch.equal(cache[pg[s // PAGE], 1, s % PAGE], self.v[t])
                after[pg[s // PAGE], :, s % PAGE] = cache[pg[s // PAGE], :, s % PAGE]
                t += 1
        assert torch.equal(cache, after)


ROWS = [(1, 1), (40, 17), (16, 16), (300, 1), (0, 0), (33, 0), (70, 3)]


def make(rot_dim, interleaved, **scaling):
    return K.rotary(rot_dim, interleaved=interleaved, device=DEV, **scaling), K.rotary_frequencies(rot_dim, **scaling)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rot_dim", [128, 64, 32, 96, 2, 6, 30, 50, 126])
@pytest.mark.parametrize("norm", [False, True])
def test_layouts(rot_dim, interleaved, dtype, norm):
    s = Step(12, 2, ROWS, dtype, seed=rot_dim, norm=norm)
    rot, (freqs, factor) = make(rot_dim, interleaved, rope_theta=1e4)
    (wq, sq), (wk, sk) = s.want(freqs, factor, interleaved)
    q, cache = s.append(rot)
    check(q, wq, sq)
    s.check_cache(cache, wk, sk)
    q2, k2 = s.rope(rot)
    assert torch.equal(q2, q)
    check(k2, wk, sk)


@pytest.mark.parametrize("scaling", [dict(rope_scale=4.0), dict(rope_scale=8.0, low_freq_factor=1.0, high_freq_factor=4.0, old_context_len=8192.0),
                                     dict(rope_scale=16.0, old_context_len=8192.0, scaling="yarn"), dict(rope_scale=8.0, scaling="ntk")])
@pytest.mark.parametrize("hq,hkv", [(32, 8), (28, 4), (40, 8), (5, 1), (3, 3), (70, 10)])
def test_scalings_at_far_positions(scaling, hq, hkv):
    s = Step(hq, hkv, [(20, 20), (9, 1), (50, 7)], seed=3, first=[131072 - 10, 2 ** 31 - 5, 1000003])
    rot, (freqs, factor) = make(128, False, rope_theta=5e5, **scaling)
    (wq, sq), (wk, sk) = s.want(freqs, factor, False)
    q, cache = s.append(rot)
    check(q, wq, sq)
    s.check_cache(cache, wk, sk)


@pytest.mark.parametrize("tokens", [1, 3, 100, 1300])
def test_sizes(tokens):
    """From blocks over a token's heads to one block a token."""
    s = Step(40, 8, [(tokens + 5, tokens)], "fp16", seed=4)
    rot, (freqs, factor) = make(128, False)
    (wq, sq), (wk, sk) = s.want(freqs, factor, False)
    q, k = s.rope(rot)
    check(q, wq, sq)
    check(k, wk, sk)
    qa, cache = s.append(rot)
    assert torch.equal(qa, q)
    keys = cache[torch.tensor(s.pages[0], device=DEV)][:, 0].reshape(-1, 8, D)[5:tokens + 5]
    assert torch.equal(keys, k)


def test_many_rows():
    rows = [(n % 40 + 1, 1 if n % 3 else 0) for n in range(300)]
    s = Step(12, 2, rows, seed=5)
    rot, (freqs, factor) = make(64, True)
    (wq, sq), (wk, sk) = s.want(freqs, factor, True)
    q, cache = s.append(rot)
    check(q, wq, sq)
    s.check_cache(cache, wk, sk)


def test_norm_alone_and_nothing():
    s = Step(12, 2, ROWS, seed=6)
    (wq, sq), (wk, sk) = s.want([], 1.0, False)
    q, k = s.rope(None)
    check(q, wq, sq)
    check(k, wk, sk)
    s = Step(12, 2, ROWS, seed=6, norm=False)
    q, k = s.rope(None)
    assert torch.equal(q, s.q) and torch.equal(k, s.k)


def test_frequencies_as_they_are():
    s = Step(12, 2, ROWS, seed=7)
    freqs = [0.0, -0.3, 2 * math.pi * 5.25, 1e-9, 3.0]
    rot = K.rotary(10, device=DEV, frequencies=freqs, factor=-1.5)
    (wq, sq), _ = s.want(freqs, -1.5, False)
    check(s.rope(rot)[0], wq, sq)


@pytest.mark.parametrize("rot_dim", [128, 50])
def test_in_place(rot_dim):
    for interleaved in (False, True):
        s = Step(12, 2, ROWS, seed=8)
        rot, _ = make(rot_dim, interleaved)
        q, k = s.rope(rot)
        cache = s.append(rot)[1]
        sc = s.cache.clone()
        K.qk_norm_rope_append(s.q, s.k, s.v, s.ip, s.off, sc, *s.tables, rot, **s.w, q_out=s.q)
        assert torch.equal(s.q, q) and torch.equal(sc, cache)
        s = Step(12, 2, ROWS, seed=8)
        s.rope(rot, q_out=s.q, k_out=s.k)
        assert torch.equal(s.q, q) and torch.equal(s.k, k)


def test_sizes_of_values():
    """Heads of zeros, of the type's smallest and largest values; NaN and infinity stay in their heads."""
    for dtype in ("bf16", "fp16"):
        s = Step(12, 2, ROWS, dtype, seed=9)
        s.q[0, 0] = 0.0
        s.q[1, 1] = torch.finfo(DT[dtype]).tiny
        s.q[2, 2] *= 100.0
        rot, (freqs, factor) = make(128, False)
        (wq, sq), _ = s.want(freqs, factor, False)
        q, _ = s.rope(rot)
        check(q, wq, sq)
        s.q[3, 3, 7], s.q[4, 4, 100] = math.nan, math.inf
        q2, _ = s.rope(rot)
        assert q2[3, 3].isnan().all() and not q2[4, 4].isfinite().all()
        q2[3, 3], q2[4, 4] = q[3, 3], q[4, 4]
        assert torch.equal(q2, q)


def test_tokens_of_no_row_stay():
    s = Step(12, 2, ROWS, seed=10, pad=6)
    rot, (freqs, factor) = make(128, True)
    (wq, sq), (wk, sk) = s.want(freqs, factor, True)
    q_out = torch.full((s.T + 6, 12, D), 3.0, dtype=torch.bfloat16, device=DEV)
    cache = s.append(rot, q_out=q_out)[1]
    check(q_out[:s.T], wq, sq)
    assert (q_out[s.T:] == 3.0).all()
    s.check_cache(cache, wk, sk)


def test_tokens_without_a_slot_append_nothing():
    s = Step(12, 2, ROWS, seed=11)
    rot, (freqs, factor) = make(128, False)
    (wq, sq), _ = s.want(freqs, factor, False)
    for bad in (-1, s.cache.shape[0], 2 ** 31 - 1):
        ids = torch.full_like(s.tables[0], bad)
        cache = s.cache.clone()
        q = K.qk_norm_rope_append(s.q, s.k, s.v, s.ip, s.off, cache, ids, *s.tables[1:], rot, **s.w)
        check(q, wq, sq)
        assert torch.equal(cache, s.cache)
    short = torch.zeros_like(s.tables[1])  # rows without pages
    cache = s.cache.clone()
    q = K.qk_norm_rope_append(s.q, s.k, s.v, s.ip, s.off, cache, s.tables[0], short, s.tables[2], rot, **s.w)
    check(q, wq, sq)
    assert torch.equal(cache, s.cache)


def test_interleaved_is_the_plain_rotation():
    """Without norms, the whole head interleaved: ``rope_append`` (whose angles are fp32) at near positions."""
    s = Step(12, 2, ROWS, "fp16", seed=12, norm=False)
    rot, (freqs, factor) = make(128, True, rope_theta=1e4)
    (wq, sq), _ = s.want(freqs, factor, True)
    old = K.rope_append(s.q, s.k, s.v, s.ip, s.off, s.cache.clone(), *s.tables, rope_theta=1e4)
    check(old, wq, sq * 64)  # an angle of up to 300 in fp32: 2^-16
    check(s.append(rot)[0], wq, sq)


def test_cache_offsets_past_32_bits():
    s = Step(32, 8, [(20, 20)], seed=13)
    rot, (freqs, factor) = make(128, False)
    (_, _), (wk, sk) = s.want(freqs, factor, False)
    cache = torch.zeros(66100, 2, PAGE, 8, D, dtype=torch.bfloat16, device=DEV)
    K.qk_norm_rope_append(s.q, s.k, s.v, s.ip, s.off, cache, i32([66099, 66000]), *s.tables[1:], rot, **s.w)
    check(cache[66099, 0], wk[:16], sk[:16])
    check(cache[66000, 0, :4], wk[16:], sk[16:])
    assert torch.equal(cache[66000, 1, :4], s.v[16:]) and not cache[66000, :, 4:].any() and not cache[:66000].any()


@torch.inference_mode()  # as the engine captures: torch's graph state must not change mode between captures
def test_graphs_and_streams():
    s = Step(28, 4, ROWS, seed=14)
    rot, _ = make(128, False)
    want, wcache = s.append(rot)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q, cache = s.append(rot)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(q, want) and torch.equal(cache, wcache)
    cache, q_out, g = s.cache.clone(), torch.empty_like(want), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        s.append(rot, cache=cache, q_out=q_out)
    for _ in range(3):
        cache.copy_(s.cache)
        q_out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(q_out, want) and torch.equal(cache, wcache)
        assert torch.equal(s.append(rot)[0], want)


def plain_attention(q, keys, vals, pos, window, cap):
    """One row's attention in 64 bits: q [T, hq, 128] at positions pos over keys, vals [n, hkv, 128]."""
    G = q.shape[1] // keys.shape[1]
    k, v = (x.double().repeat_interleave(G, 1).transpose(0, 1).contiguous() for x in (keys, vals))
    z = torch.matmul(q.double().transpose(0, 1).contiguous(), k.transpose(1, 2).contiguous()) / math.sqrt(D)
    z = cap * torch.tanh(z / cap)
    at = torch.arange(keys.shape[0], device=DEV)
    hidden = (at > pos[:, None]) | (at <= pos[:, None] - window)
    z = z.masked_fill(hidden, -math.inf)
    p = torch.softmax(z, -1)
    return torch.matmul(p, v).transpose(0, 1), torch.matmul(p, v.abs()).transpose(0, 1)


@pytest.mark.parametrize("window", [50, 1 << 20])
def test_a_layer_as_it_is_used(window):
    """Two chunks of a prompt, then single tokens: each step's norms, rotation and append, then attention over the cache
    it left.  The attention is checked over the keys that the steps appended, those against their own 64-bit values."""
    hq, hkv, cap, total = 12, 2, 20.0, 130
    g = torch.Generator(device=DEV)
    g.manual_seed(15)
    lens = [total, 77]
    order = torch.randperm(20, generator=torch.Generator().manual_seed(15)).tolist()
    cache = torch.full((20, 2, PAGE, hkv, D), math.nan, dtype=torch.bfloat16, device=DEV)
    table = [order[:9], order[9:14]]
    w = {n: torch.empty(D, dtype=torch.bfloat16, device=DEV).normal_(1, 0.3, generator=g) for n in ("q_weight", "k_weight")}
    rot, (freqs, factor) = make(96, False, rope_theta=1e4, rope_scale=4.0, old_context_len=64.0, scaling="yarn")
    rule = K.ScoreRule(softcap=cap, window=window)
    have = [0, 0]
    vals = [[], []]
    for step in ([60, 41], [66, 33], [1, 1], [1, 1], [2, 1]):
        T = sum(step)
        qkv = torch.empty(T, (hq + 2 * hkv) * D, dtype=torch.bfloat16, device=DEV).normal_(0, 2, generator=g)
        q, k, v = (x.unflatten(-1, (-1, D)) for x in qkv.split([hq * D, hkv * D, hkv * D], -1))
        now = [h + n for h, n in zip(have, step)]
        counts = [-(-n // PAGE) for n in now]
        tables = (i32([p for t, c in zip(table, counts) for p in t[:c]]), i32(indptr(counts)), i32([(n - 1) % PAGE + 1 for n in now]))
        ip, off = i32(indptr(step)), i32(have)
        qr = K.qk_norm_rope_append(q, k, v, ip, off, cache, *tables, rot, **w)
        kv_ip = (tables[1], tables[0], tables[2])
        if max(step) == 1:
            o = K.paged_decode_rule(qr, cache, *kv_ip, rule, max_pages_per_row=max(counts))
            same = K.paged_prefill_rule(qr, cache, ip, *kv_ip, rule, max_qo_len=1)
            assert (same.double() - o.double()).abs().max() <= 0.1
        else:
            o = K.paged_prefill_rule(qr, cache, ip, *kv_ip, rule, max_qo_len=max(step))
        t = 0
        for r, n in enumerate(step):
            pos = torch.arange(have[r], now[r], device=DEV)
            wk, sk = turned(k[t:t + n], w["k_weight"], 1e-6, freqs, factor, pos.tolist(), False)
            row = cache[torch.tensor(table[r], device=DEV)].transpose(0, 1).reshape(2, -1, hkv, D)[:, :now[r]]
            check(row[0, have[r]:], wk, sk)
            vals[r].append(v[t:t + n])
            assert torch.equal(row[1], torch.cat(vals[r]))
            want, A = plain_attention(qr[t:t + n], row[0], row[1], pos, window, cap)
            # u of each p and of o; scores of |x| <= 20 (the cap) from sums of |q k| <= 150: 2^-17 150 + 2^-20 20
            tol = A * (2.0 ** -8 + 2 * 1.2e-3) + want.abs() * 2.0 ** -8
            assert ((o[t:t + n].double() - want).abs() <= tol).all()
            t += n
        have = now
    assert lens[0] == have[0] and lens[1] == have[1]
