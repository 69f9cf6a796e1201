"""The engine serving rows that share pages: requests of one prefix, forks, and captured decode steps over shared pages.

tiny-test has 2 kv heads, so sharing pays (8192 page-heads spared) from 16 rows of 274 common pages on: the rows here
share 4800 tokens, 300 pages.
"""
import pytest
import torch

import delta_amd.kernels as K
from oracle import delta_oracle as O
from test_gpu_engine import _csr, _restore, _snapshot, assert_close, make_engine

pytestmark = pytest.mark.gpu
SCALE = 1 / 128 ** 0.5
PREFIX = 4800


@pytest.fixture
def calls(monkeypatch):
    """Calls of the shared launches."""
    n = {"paged_decode_prefix": 0, "paged_prefill_prefix": 0, "copy_pages": 0}
    for name in n:
        def counted(*a, _f=getattr(K, name), _n=name, **kw):
            n[_n] += 1
            return _f(*a, **kw)
        monkeypatch.setattr(K, name, counted)
    return n


def prompt(n, seed):
    return torch.randint(1, 250, (n,), generator=torch.Generator().manual_seed(seed))


def check_decode_layer(layer, rows, what):
    """The layer's last recorded (q, o) of a decode step against the oracle; rows: slot -> (pages, cached tokens)."""
    q, o = layer.attention.record[-1]
    cache = layer.attention.kv_cache.kv_cache.cpu()
    for s, (pages, n) in rows.items():
        use = torch.tensor(pages[:(n + 15) // 16], dtype=torch.int32)
        ref, _ = O.paged_decode_attention(q[s:s + 1].cpu(), cache, torch.tensor([0, len(use)], dtype=torch.int32), use,
                                          torch.tensor([(n - 1) % 16 + 1], dtype=torch.int32), SCALE)
        assert_close(o[s:s + 1], ref, f"{what} slot {s}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_captured_steps_over_shared_pages(dtype, calls):
    lens = [PREFIX + 20 * i for i in range(16)]  # slot 0 owns nothing but its next page
    eng = make_engine(graph=True, B=16, max_len=5376, dtype=dtype)
    eng.prepare_synthetic_decode(lens, decode_budget=40, seed=5, shared_tokens=PREFIX + 3)
    assert eng._sharing
    bt = eng.slot_block_table.cpu()
    assert (bt[:, :300] == bt[0, :300]).all() and len(set(bt[:, 300].tolist())) == 16
    snap = _snapshot(eng)
    for layer in eng.model.layers:
        layer.attention.record = []
    eager = [eng.decode_steps(1, use_graph=False).clone()]
    assert calls["paged_decode_prefix"] == sum(r == "full" for r in eng.layer_roles) > 0
    ip, ind, last, _ = _csr(eng)
    for li, (role, layer) in enumerate(zip(eng.layer_roles, eng.model.layers)):
        if role == "full":
            (q, o), = layer.attention.record
            ref, _ = O.paged_decode_attention(q.cpu(), layer.attention.kv_cache.kv_cache.cpu(), ip, ind, last, SCALE)
            assert_close(o, ref, f"layer {li}")
        layer.attention.record = None
    eager += [eng.decode_steps(1, use_graph=False).clone() for _ in range(19)]
    eager_caches = [l.attention.kv_cache.kv_cache.clone() for l in eng.model.layers]
    _restore(eng, snap)
    for i in range(20):
        tok = eng.decode_steps(1, use_graph=True).clone()
        a = torch.randn(256, 256, device=eng.device)
        (a @ a).sum().item()  # unrelated eager work between replays
        assert torch.equal(tok, eager[i]), f"replay {i}"
    assert eng._decode_graph_stats["replays"] == 20 and eng._decode_graph_failed is None
    for l, c in zip(eng.model.layers, eager_caches):
        assert torch.equal(l.attention.kv_cache.kv_cache, c)
    # rows of their own again: the ordinary launches, captured anew
    n = calls["paged_decode_prefix"]
    eng.prepare_synthetic_decode(lens, decode_budget=40, seed=5)
    assert not eng._sharing and eng._decode_graph is None
    eng.decode_steps(3, use_graph=True)
    assert calls["paged_decode_prefix"] == n
    # and other rows sharing other pages, through the tables that a captured step reads
    eng.prepare_synthetic_decode(lens, decode_budget=40, seed=6, shared_tokens=PREFIX)
    assert eng._sharing
    eng.decode_steps(2, use_graph=True)
    assert calls["paged_decode_prefix"] > n


def test_too_few_shared_pages_take_the_ordinary_launches(calls):
    eng = make_engine(B=16, max_len=5376)
    eng.prepare_synthetic_decode([PREFIX] * 16, decode_budget=16, seed=5, shared_tokens=272 * 16)
    assert not eng._sharing
    eng.decode_steps(1, use_graph=False)
    assert calls["paged_decode_prefix"] == 0
    with pytest.raises(ValueError, match="cannot share"):
        eng.prepare_synthetic_decode([100] * 16, decode_budget=16, shared_tokens=112)


@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graph"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_requests_of_one_prefix(dtype, graph, calls):
    """Twenty requests through 16 slots: the prompts' K/V are those of an engine that shares nothing, the decode steps'
    attention is the oracle's, and every page goes back."""
    prefix = prompt(PREFIX + 5, 0)  # five tokens behind the last whole page: every request's own
    own = [prompt(0 if i == 3 else 1 + 7 * i, i) for i in range(20)]
    caps = [PREFIX + 160 + i for i in range(20)]
    eng = make_engine(B=16, max_len=5120, dtype=dtype, graph=graph)
    eng.add_requests(own, caps, [], prefix_ids=prefix)
    kv, seen = {}, [0]

    def rows_kv(e, req, n):
        pages = torch.tensor(req.pages[:n // 16], device=e.device)  # whole pages: what lies behind the last token differs
        return [e.model.layers[li].attention.kv_cache.kv_cache[pages].float().cpu() for li in (0, -1)]

    def on_step(e, i):
        for s in e.scheduler.occupied():
            req = e.scheduler.request_in(s)
            if len(req.generated) == 1 and req.rid in (0, 3, 15):
                kv[req.rid] = rows_kv(e, req, len(req.prompt))
        layer = e.model.layers[0]
        if layer.attention.record and not graph and seen[0] < 3 and layer.attention.record[-1][0].shape[0] == 16:
            live = {s: e.scheduler.request_in(s) for s in e.scheduler.occupied()}
            if all(len(r.generated) > 1 and not r.finished for r in live.values()):
                check_decode_layer(layer, {s: (r.pages, r.kv_len()) for s, r in list(live.items())[::5]}, f"step {i}")
                seen[0] += 1
        layer.attention.record = [] if not graph else None

    if not graph:
        eng.model.layers[0].attention.record = []
    results = eng.run_scheduler_loop(on_step=on_step)
    assert len(results) == 20 and eng.page_pool.available == eng.page_pool.total_pages
    for r, p, cap in zip(results, own, caps):
        assert r["output_length"] == cap - PREFIX - 5 - len(p)
    assert graph or seen[0] == 3
    assert calls["paged_decode_prefix"] > 0 and calls["paged_prefill_prefix"] > 0
    assert not graph or (eng._decode_graph_stats["replays"] > 0 and eng._decode_graph_failed is None)
    assert not eng._sharing  # nothing is being served

    alone = make_engine(B=3, max_len=5120, dtype=dtype)
    alone.add_requests([torch.cat([prefix, own[i]]) for i in (0, 3, 15)], PREFIX + 160, [])
    want = {}

    def first(e, i):
        if not want:
            want.update({rid: rows_kv(e, e.scheduler.requests[j], len(e.scheduler.requests[j].prompt))
                         for j, rid in enumerate((0, 3, 15))})

    alone.run_scheduler_loop(on_step=first)
    for rid in (0, 3, 15):
        for a, b in zip(kv[rid], want[rid]):
            cos = torch.nn.functional.cosine_similarity(a.flatten(), b.flatten(), dim=0).item()
            assert cos > 0.999, (rid, cos)


@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graph"])
def test_forks(graph, calls):
    """A request branches into fifteen others while it decodes, and one of those once more; their attention is the
    oracle's over their own pages, the copied tokens are the parent's, and the parent may end first."""
    eng = make_engine(B=16, max_len=5120, graph=graph)
    eng.add_requests([prompt(PREFIX + 7, 1)], PREFIX + 40, [])
    tails, checked = [], [0]

    def tail(page, n):
        return [l.attention.kv_cache.kv_cache[page, :, :n].clone() for l in eng.model.layers]

    def on_step(e, i):
        reqs = e.scheduler.requests
        r = reqs[0]
        if i == 5:
            for j in range(14):
                rid = e.fork_request(0, prompt(1 + j % 3, j), max_length=PREFIX + 60 + j)
                c = reqs[rid]
                assert c.pages[:300] == r.pages[:300] and 0 < c.fill == r.fill
                for a, b in zip(tail(r.pages[-1], r.fill), tail(c.pages[-1], c.fill)):
                    assert torch.equal(a, b)
                tails.append((rid, c.pages[-1], tail(c.pages[-1], c.fill)))
        if i == 8:
            child = reqs[2]
            rid = e.fork_request(2, torch.tensor([], dtype=torch.long), max_length=PREFIX + 70, eot_token_ids=[])
            assert reqs[rid].prompt.tolist() == child.prompt.tolist() + child.generated
            assert reqs[rid].pages[:300] == r.pages[:300]
            with pytest.raises(RuntimeError, match="no free slot"):
                e.fork_request(0, torch.tensor([1]))
            assert e._sharing
        if i > 5:
            for rid, page, want in tails:  # what the parent cached stays in the copies
                if not reqs[rid].finished and page in reqs[rid].pages:
                    for a, b in zip(tail(page, want[0].shape[1]), want):
                        assert torch.equal(a, b)
        layer = e.model.layers[0]
        if not graph:
            live = {s: e.scheduler.request_in(s) for s in e.scheduler.occupied()}
            if i in (7, 11, 50) and all(len(x.generated) > 1 and not x.finished for x in live.values()):
                check_decode_layer(layer, {s: (x.pages, x.kv_len()) for s, x in list(live.items())[::3]}, f"step {i}")
                checked[0] += 1
            layer.attention.record = []

    if not graph:
        eng.model.layers[0].attention.record = []
    results = eng.run_scheduler_loop(on_step=on_step)
    assert len(results) == 16 and eng.page_pool.available == eng.page_pool.total_pages
    assert all(r["status"] == "finished" for r in results)
    assert graph or checked[0] >= 2
    assert calls["copy_pages"] >= 14 and calls["paged_decode_prefix"] > 0 and calls["paged_prefill_prefix"] > 0
    assert not graph or (eng._decode_graph_stats["replays"] > 0 and eng._decode_graph_failed is None)


def test_what_cannot_be_forked_is_refused():
    eng = make_engine(B=3, max_len=256)
    eng.add_requests([prompt(20, 0), prompt(20, 1)], [40, 24], [])
    with pytest.raises(ValueError, match="no request 7"):
        eng.fork_request(7, torch.tensor([1]))
    with pytest.raises(RuntimeError, match="not decoding"):
        eng.fork_request(0, torch.tensor([1]))
    seen = []

    def on_step(e, i):
        if e.scheduler.requests[1].finished and not seen:
            seen.append(i)
            pages = e.page_pool.available
            with pytest.raises(RuntimeError, match="not decoding"):
                e.fork_request(1, torch.tensor([1]))
            with pytest.raises(ValueError, match="max_length"):
                e.fork_request(0, prompt(30, 2))
            with pytest.raises(ValueError, match="max_length"):
                e.fork_request(0, prompt(3, 2), max_length=300)
            with pytest.raises(ValueError, match="1-D"):
                e.fork_request(0, torch.tensor([[1]]))
            assert e.page_pool.available == pages and len(e.scheduler.requests) == 2

    eng.run_scheduler_loop(on_step=on_step)
    assert seen and eng.page_pool.available == eng.page_pool.total_pages
    for bad in (torch.tensor([]), torch.tensor([], dtype=torch.long), torch.tensor([[1]]), torch.tensor([1.5])):
        with pytest.raises(ValueError, match="prefix_ids"):
            eng.add_requests([prompt(4, 0)], 20, [], prefix_ids=bad)


@pytest.mark.parametrize("limit,value", [("SHARING_TOKENS", 40), ("SHARING_PAIRS", 2)])
def test_prompt_steps_of_many_tokens_take_the_ordinary_launch(limit, value, calls, monkeypatch):
    import delta_amd.backend as backend
    monkeypatch.setattr(backend, limit, value)
    eng = make_engine(B=16, max_len=5120)
    eng.add_requests([prompt(3 + i, i) for i in range(16)], PREFIX + 40, [], prefix_ids=prompt(PREFIX, 0))
    eng.run_scheduler_loop()
    assert calls["paged_prefill_prefix"] == 0 and calls["paged_decode_prefix"] > 0
    assert eng.page_pool.available == eng.page_pool.total_pages


def test_prompts_that_leave_no_room_are_refused():
    eng = make_engine(B=3, max_len=256)
    with pytest.raises(ValueError, match="no room"):
        eng.add_requests([prompt(3, 0), prompt(56, 1)], 256, [], prefix_ids=prompt(200, 2))
    assert not eng.scheduler.requests
    eng.add_requests([prompt(3, 0), prompt(55, 1)], 256, [], prefix_ids=prompt(200, 2))
    eng.run_scheduler_loop()
    assert [r.kv_len() for r in eng.scheduler.requests] == [255, 255]
    assert eng.page_pool.available == eng.page_pool.total_pages


def test_requests_added_and_forked_while_others_run():
    """A prefix group that arrives later, of which one prompt adds nothing, beside forks of a request without a prefix."""
    eng = make_engine(B=4, max_len=256, graph=True)
    eng.add_requests([prompt(30, 0)], 80, [])
    forks = []

    def on_step(e, i):
        r = e.scheduler.requests[0]
        if len(r.generated) == 3:
            e.add_requests([prompt(0, 1), prompt(9, 2), prompt(33, 3), prompt(2, 4)], 120, [], prefix_ids=prompt(48, 5))
            forks.append(e.fork_request(0, prompt(5, 6), max_length=70))

    results = eng.run_scheduler_loop(on_step=on_step)
    assert len(results) == 6 and all(r["status"] == "finished" for r in results)
    assert [len(r.prompt) + len(r.generated) for r in eng.scheduler.requests] == [80] + [120 if i != forks[0] else 70 for i in range(1, 6)]
    assert eng.page_pool.available == eng.page_pool.total_pages
