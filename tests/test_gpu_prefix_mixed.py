"""Shared-prefix attention over mixed batches: drawn tables, rows without tokens, captured prompt calls, calls that run at
the same time.  Tolerances as in test_gpu_prefix.py."""
import math
import random

import pytest
import torch

from delta_amd import kernels as K
from test_gpu_prefix import DEV, HEADS, Batch, D

pytestmark = pytest.mark.gpu


def drawn(seed, decode):
    """Rows of any kind: of no prefix, an empty one, one that nobody else has; without cached tokens, with fewer than query
    tokens, without query tokens."""
    rng = random.Random(seed)
    hq, hkv = rng.choice(HEADS)
    prefixes = [rng.choice([0, 1, 2, 3, 4, 5, 8, 17, 64, 129, 300]) for _ in range(rng.randint(0, 4))]
    rows = []
    for _ in range(rng.choice([1, 2, 3, 7, 20, 45])):
        p = rng.choice([-1] + list(range(len(prefixes))) * 3)
        qn = 1 if decode else rng.choice([0, 1, 1, 2, 5, 16, 17, 33, 70])
        rows.append((p, rng.choice([0, 1, 15, 16, 17, 63, 64, 65, rng.randint(0, 700)]), qn))
    if not any(r[2] for r in rows):
        rows[0] = (*rows[0][:2], 3)
    return Batch(hq, hkv, prefixes, rows, dtype=rng.choice(["bf16", "fp16"]), seed=seed,
                 stale=rng.choice([None, math.nan, math.inf]))


@pytest.mark.parametrize("seed", range(24))
def test_drawn_decode(seed):
    b = drawn(seed, True)
    b.check(b.decode(), b.want())


@pytest.mark.parametrize("seed", range(100, 124))
def test_drawn_prompts(seed):
    b = drawn(seed, False)
    b.check(b.prefill(), b.want())


def test_prompt_tokens_before_the_first_cached_one_attend_nothing():
    b = Batch(12, 2, [3], [(-1, 5, 9), (0, 20, 20), (-2, 0, 4), (0, 0, 7)], seed=40)
    o, lse = b.prefill()
    b.check((o, lse), b.want())
    assert (o[:4] == 0).all() and (lse[:4] == -math.inf).all()   # positions -4 .. -1
    assert (o[29:33] == 0).all() and (lse[29:33] == -math.inf).all()  # a row without pages


@pytest.mark.parametrize("bad", [-1, 10 ** 6, -(1 << 31), (1 << 31) - 1])
def test_prompt_pages_outside_the_cache_are_dropped(bad):
    b = Batch(28, 4, [9], [(0, 70, 20), (0, 33, 33), (-1, 90, 40)], seed=41)
    pages = [list(p) for p in b.pages]
    b.t["prefix_indices"][4] = bad
    for r in (0, 1):
        pages[r][4] = bad
    pages[2][2] = bad
    b.t["kv_indices"][:sum(map(len, pages))] = torch.tensor([x for p in pages for x in p], dtype=torch.int32, device=DEV)
    b.check(b.prefill(), b.want(tables=pages))


@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.0])
def test_prompt_scales(scale):
    """(2.0: sum |q_i k_i| scale is about 128 * 0.08 * 0.8 * 2 = 16, so a score is off by 128 * 2^-24 * 16 = 1.2e-4.)"""
    b = Batch(32, 8, [20], [(0, 30, 7), (0, 3, 3), (-1, 60, 40)], seed=42)
    b.q *= 0.1
    b.check(b.prefill(sm_scale=scale), b.want(scale=scale))


def test_prompt_strided_q_and_out():
    b = Batch(12, 4, [11], [(0, 40, 9), (0, 3, 3), (-1, 60, 30)], seed=43)
    wide = torch.randn(42, 2, 14, D, device=DEV).to(torch.bfloat16)
    q = wide[:, 1, 1:13]
    q.copy_(b.q)
    out = torch.zeros(42, 15, D + 8, dtype=torch.bfloat16, device=DEV)[:, 2:14, 2:2 + D]
    b.check(b.prefill(q=q, out=out), b.want())
    assert (out._base[:, :2] == 0).all() and (out._base[:, :, :2] == 0).all() and (out._base[:, :, 2 + D:] == 0).all()


def test_captured_prompts_follow_tables_and_queries():
    b = Batch(12, 2, [30, 11], [(0, 20, 5), (1, 33, 30), (0, 50, 1), (-1, 60, 20)], seed=44)
    ws = torch.empty(K.prefix_attention_workspace_bytes(56, 12, 2, b.t["kv_indices"].numel()), dtype=torch.uint8, device=DEV)
    out, lse = torch.zeros_like(b.q), torch.zeros(56, 12, device=DEV)
    b.prefill(out=out, lse=lse, workspace=ws)
    torch.cuda.synchronize()
    qo = torch.tensor(b.qo, dtype=torch.int32, device=DEV)
    t = b.t
    g = torch.cuda.CUDAGraph()
    with torch.inference_mode(), torch.cuda.graph(g):
        K.paged_prefill_prefix(b.q, b.cache, qo, t["kv_indptr"], t["kv_indices"], t["last"], t["row_prefix"], t["prefix_indptr"],
                               t["prefix_indices"], max_qo_len=30, out=out, lse=lse, workspace=ws)
    for i in range(4):
        if i == 2:  # two rows lose their prefix: the same context from their own CSR
            t["row_prefix"].copy_(torch.tensor([-1, 1, -1, -1], dtype=torch.int32))
        b.q.normal_(0, 1)
        out.fill_(9.0)
        lse.fill_(9.0)
        g.replay()
        torch.cuda.synchronize()
        b.check((out, lse), b.want())
        torch.randn(64, 64, device=DEV).sum().item()


@pytest.mark.parametrize("table", ["kv_indptr", "prefix_indptr", "qo"])
def test_tables_that_do_not_ascend_write_nothing_out_of_place(table):
    b = Batch(12, 2, [9, 4], [(0, 20, 3), (1, 33, 30), (0, 50, 1), (-1, 60, 20)], seed=49)
    want = b.want()
    good = (b.t[table].clone() if table != "qo" else list(b.qo))
    if table == "qo":
        b.qo = [0, 33, 3, 34, 54]
    elif table == "kv_indptr":
        b.t[table][1:3] = b.t[table][1:3].flip(0)
    else:
        b.t[table].copy_(torch.tensor([9, 0, 13], dtype=torch.int32))
    room, lse = torch.full((60, 12, D), 3.0, dtype=torch.bfloat16, device=DEV), torch.full((60, 12), 4.0, device=DEV)
    cache = b.cache.clone()
    K.paged_prefill_prefix(b.q, b.cache, torch.tensor(b.qo, dtype=torch.int32, device=DEV), b.t["kv_indptr"], b.t["kv_indices"],
                           b.t["last"], b.t["row_prefix"], b.t["prefix_indptr"], b.t["prefix_indices"], max_qo_len=33,
                           out=room[3:57], lse=lse[3:57])
    torch.cuda.synchronize()
    for x, v in ((room, 3), (lse, 4)):
        assert (x[:3] == v).all() and (x[57:] == v).all()
    assert torch.equal(b.cache, cache)
    if table == "qo":
        b.qo = good
    else:
        b.t[table].copy_(good)
    b.check(b.prefill(), want)


def test_two_graphs_share_a_workspace():
    """Replayed in turn on one stream; nothing of one call is kept for the next."""
    bs = [Batch(32, 8, [40], [(0, 30 + i, 1) for i in range(9)], seed=45), Batch(12, 2, [7, 90], [(i % 2, 17 * i, 1) for i in range(20)], seed=46)]
    ws = torch.empty(max(K.prefix_attention_workspace_bytes(len(b.rows), b.hq, b.hkv, 8192) for b in bs), dtype=torch.uint8, device=DEV)
    ws.fill_(255)
    calls = []
    for b in bs:
        out, lse = torch.zeros_like(b.q), torch.zeros(len(b.rows), b.hq, device=DEV)
        g = torch.cuda.CUDAGraph()
        b.decode(out=out, lse=lse, workspace=ws)
        torch.cuda.synchronize()
        with torch.inference_mode(), torch.cuda.graph(g):
            b.decode(out=out, lse=lse, workspace=ws)
        calls.append((g, out, lse, b.want()))
    for i in (0, 1, 1, 0, 1, 0):
        g, out, lse, want = calls[i]
        out.fill_(9.0)
        g.replay()
        torch.cuda.synchronize()
        bs[i].check((out, lse), want)
        torch.randn(64, 64, device=DEV).sum().item()


def test_calls_at_the_same_time():
    bs = [Batch(32, 8, [300], [(0, 1 + 37 * i % 300, 1) for i in range(33)], seed=47),
          Batch(28, 4, [200, 5], [(i % 2, 11 + 5 * i, 11) for i in range(12)], seed=48)]
    want = [bs[0].decode(), bs[1].prefill()]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, f in enumerate((bs[0].decode, bs[1].prefill)):
            with torch.cuda.stream(streams[i]):
                got[i].append(f())
    torch.cuda.synchronize()
    for w, rs in zip(want, got):
        for r in rs:
            assert torch.equal(r[0], w[0]) and torch.equal(r[1], w[1])


def test_rows_behind_the_tables_end_are_empty():
    """A batch padded with rows of zero bounds: their o is 0, the others' unchanged."""
    b = Batch(28, 4, [9, 4], [(0, 20, 1), (1, 33, 1), (-1, 60, 1)], seed=50)
    o, lse = b.decode()
    pad = lambda t, n: torch.cat([t, torch.zeros(n, dtype=torch.int32, device=DEV)])
    t = b.t
    q = torch.cat([b.q, torch.randn(4, 28, D, device=DEV).to(b.q.dtype)])
    lse2 = torch.zeros(7, 28, device=DEV)
    o2 = K.paged_decode_prefix(q, b.cache, pad(t["kv_indptr"], 4), t["kv_indices"], pad(t["last"], 4), pad(t["row_prefix"], 4),
                               pad(t["prefix_indptr"], 3), t["prefix_indices"], max_pages_per_row=8192, lse=lse2)
    b.check((o2[:3], lse2[:3]), b.want())
    assert (o2[3:] == 0).all() and (lse2[3:] == -math.inf).all()
