"""The engine's bookkeeping of shared pages without a GPU: an ``LMBackend`` on CPU tables whose model steps are stand-ins."""
from types import SimpleNamespace

import pytest
import torch

import delta_amd.backend as backend
from delta_amd.backend import LMBackend
from delta_amd.scheduler import BatchSlots, PagePool

PAGE = 16


@pytest.fixture
def host_engine(monkeypatch):
    """An engine of ``batch`` slots whose forward hands every active request one token (its prompt is cached by then)."""
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)

    def make(batch=16, pages=337, hq=4, hkv=2):
        e = LMBackend.__new__(LMBackend)
        e.device, e.batch_size, e.pages_per_slot, e.max_length = torch.device("cpu"), batch, pages, (pages - 1) * PAGE
        e.model = SimpleNamespace(config=SimpleNamespace(n_head=hq, n_local_heads=hkv), layers=[])
        e.max_num_pages = batch * pages
        e.page_pool = PagePool(e.max_num_pages, seed=0)
        e.scheduler = BatchSlots(batch, e.page_pool, verbose=False)
        e.scratch_pages = torch.arange(e.max_num_pages, e.max_num_pages + batch, dtype=torch.int32)
        e.slot_block_table = e.scratch_pages[:, None].repeat(1, pages)
        e.cachelens, e.active = torch.zeros(batch, dtype=torch.int32), torch.zeros(batch, dtype=torch.int32)
        e._host_lens, e._host_active, e._slot_pages = [0] * batch, [0] * batch, [pages] * batch
        e.row_prefix = torch.full((batch,), -1, dtype=torch.int32)
        e.prefix_indptr = torch.zeros(batch // 2 + 1, dtype=torch.int32)
        e.prefix_indices = torch.zeros(e.max_num_pages, dtype=torch.int32)
        e.prefix_workspace, e._sharing, e._decode_graph = None, False, None
        e.page_selector = SimpleNamespace(paged_kv_indptr=None, paged_kv_indices=None, paged_kv_last_page_len=None)
        e.enable_delta_impl_profile = e.throughput_mode = e.is_main_process = False
        e.tokenizer, e._step = None, None
        e.enable_selective_cache, e.layer_roles = False, ["full"] * 4
        e.seen = []

        def forward(i):
            for s in e.scheduler.occupied():
                r = e.scheduler.request_in(s)
                old = len(r.pages)
                r.reserve(len(r.next_input()))
                e._sync_slot_block_table(s, r, old)
                r.record(7)
            e.seen.append(e._sharing)

        e._forward = forward
        e._compute_prefix = lambda prefix: prefix.reserve()
        return e

    return make


def prompts(n, length=3):
    return [torch.arange(length) + i for i in range(n)]


def test_sharing_ends_with_the_last_sharers(host_engine):
    """Sixteen rows that end in one step leave no prefix to the steps that follow the loop."""
    e = host_engine()
    e.add_requests(prompts(16), 4800 + 6, [], prefix_ids=torch.arange(4800))
    e.run_scheduler_loop()
    assert any(e.seen) and e.page_pool.available == e.page_pool.total_pages
    assert not e._sharing and e._decode_csr().prefix is None


def test_a_prefix_that_could_not_be_computed_is_computed_again(host_engine):
    """A failing forward (out of memory, say) leaves no pages behind that pass for the prefix's K and V."""
    e = host_engine(batch=2)
    del e._compute_prefix
    tries = []

    def model(*a):
        tries.append(a[0].shape[1])
        if len(tries) == 1:
            raise torch.OutOfMemoryError("no room for the prefix")

    e.model = type("Model", (), {"config": e.model.config, "layers": [], "__call__": staticmethod(model)})()
    e.add_requests(prompts(3), 60, [], prefix_ids=torch.arange(40))
    px = e.scheduler.requests[0].prefix
    with pytest.raises(torch.OutOfMemoryError):
        e.run_scheduler_loop()
    assert px.pages == [] and e.page_pool.available == e.page_pool.total_pages and e._step is None
    assert e.scheduler.occupied() == [] and list(e.scheduler.waiting) == [0, 1, 2]  # as before the call
    e.run_scheduler_loop()
    assert tries == [32, 32] and all(r.finished for r in e.scheduler.requests)
    assert e.page_pool.available == e.page_pool.total_pages


def test_a_fork_whose_page_copy_fails_is_not_served(host_engine, monkeypatch):
    e = host_engine(batch=2)
    e.add_requests(prompts(1, 5), 60, [])

    def refuse(*a, **kw):
        raise torch.OutOfMemoryError("no room for the tables")

    monkeypatch.setattr(backend.K, "copy_pages", refuse)
    tries = []

    def on_step(e, i):
        if i == 3:
            pages = e.page_pool.available
            with pytest.raises(torch.OutOfMemoryError):
                e.fork_request(0, torch.tensor([1, 2]))
            tries.append(i)
            assert e.page_pool.available == pages and len(e.scheduler.requests) == 1 and e.scheduler.occupied() == [0]

    e.run_scheduler_loop(on_step=on_step)
    assert tries and e.page_pool.available == e.page_pool.total_pages


def test_prompt_steps_go_on_where_the_partials_find_no_room(host_engine, monkeypatch):
    """As ``paged_prefill`` does: the ordinary launch attends the same tables."""
    e = host_engine()
    calls = []

    def shared(*a, **kw):
        calls.append("shared")
        raise torch.OutOfMemoryError("no room for the partials")

    def ordinary(q, cache, *tables, **kw):
        calls.append("ordinary")
        return q, tables, kw["max_qo_len"]

    monkeypatch.setattr(backend.K, "paged_prefill_prefix", shared)
    monkeypatch.setattr(backend.K, "paged_prefill", ordinary)
    e.workspace = None
    e._step = backend._StepCSR("prefill", "ip", "ind", "last", 7, qo_indptr="qo", max_qo=5, single_pages=[], prefix=(1, 2, 3))
    assert e.attn_full("q", "cache") == ("q", ("qo", "ip", "ind", "last"), 5)
    assert e.attn_full("q", "cache") == ("q", ("qo", "ip", "ind", "last"), 5)  # the next layer does not try again
    assert calls == ["shared", "ordinary", "ordinary"]


def test_decode_steps_go_on_where_the_workspace_finds_no_room(host_engine, monkeypatch):
    e = host_engine()
    rows = {s: list(range(300)) + [300 + s] for s in range(16)}
    empty = torch.empty

    def full(*a, **kw):
        if kw.get("dtype") is torch.uint8:
            raise torch.OutOfMemoryError("no room for the workspace")
        return empty(*a, **kw)

    monkeypatch.setattr(torch, "empty", full)
    e._update_sharing(rows)
    assert not e._sharing and e._decode_csr().prefix is None
    monkeypatch.setattr(torch, "empty", empty)
    e._update_sharing(rows)
    assert e._sharing and e.prefix_workspace is not None


def step(sharers, prefix_pages, longs=()):
    """Rows of a prompt step: (own cached tokens, new tokens) behind a prefix of so many pages, and beside it rows of none."""
    pages, qo, lens, at = [], [], [], prefix_pages
    for own, q in list(sharers) + list(longs):
        shared = prefix_pages if len(pages) < len(sharers) else 0
        n = -(-(own + q) // PAGE)
        pages.append(list(range(shared)) + list(range(at, at + n)))
        at += n
        qo.append(q)
        lens.append(shared * PAGE + own + q)
    return pages, qo, lens


@pytest.mark.parametrize("heads,rows,shared", [  # us shared / ordinary
    ((32, 8), step([(40, 1)] * 31, 300), True),                    # 25 / 59
    ((32, 8), step([(40, 1)] * 31, 600, [(0, 1100)]), True),       # 52 / 156
    ((32, 8), step([(40, 1)] * 31, 600, [(0, 2000)]), True),       # 98 / 179
    ((32, 8), step([(40, 1)] * 31, 300, [(0, 4000)]), False),      # 264 / 200
    ((32, 8), step([(40, 1)] * 31, 600, [(0, 8000)]), False),      # 906 / 618
    ((32, 8), step([(20, 20)] * 31, 300, [(0, 4000)]), False),     # 300 / 225
    ((32, 8), step([(0, 20)] * 31, 300, [(0, 2000)] * 4), False),  # 341 / 244
    ((28, 4), step([(40, 1)] * 31, 600, [(0, 4000)]), False),      # 237 / 190
    ((12, 2), step([(40, 1)] * 31, 600, [(0, 8000)]), False),      # 365 / 252
    ((12, 2), step([(40, 1)] * 15, 1000, [(0, 2000)]), True),      # 55 / 94
    ((32, 8), step([(0, 60)] * 8, 400), True),                     # 86 / 140
    ((32, 8), step([(0, 20)] * 32, 400), True),                    # 105 / 138
    ((32, 8), step([(0, 60)] * 64, 400), False),                   # 475 / 398
    ((32, 8), step([(0, 250)] * 64, 200), False),                  # 1026 / 868
    ((32, 8), step([(0, 20)] * 64, 50), False),                    # 61 / 33
    ((28, 4), step([(0, 60)] * 64, 100), False),                   # 169 / 117
])
def test_prompt_steps_share_where_that_is_faster(host_engine, heads, rows, shared):
    """Rows that gain nothing from sharing weigh against those that do: one launch attends them all."""
    pages, qo, lens = rows
    e = host_engine(batch=len(qo), hq=heads[0], hkv=heads[1])
    assert (e._prompt_prefixes(pages, qo, lens) is not None) == shared


@pytest.mark.parametrize("rows,heads,capacity,shared,on", [  # us a layer more (-: less) in captured steps that share
    (8, (32, 8), 9000, 147, False),   # +4.0 to -0.5 over own parts of 20 to 3000 tokens
    (8, (32, 8), 9000, 293, True),    # -0.2 to -2.8
    (16, (32, 8), 9000, 69, False),   # +2.0 to +5.2
    (16, (32, 8), 9000, 205, True),   # -1.8 to -6.2
    (32, (32, 8), 5000, 50, False),   # +3.6 to +9.3
    (32, (32, 8), 5000, 130, True),   # -7.8 at 166, +2.2 to -3.8 at 100
    (64, (32, 8), 5000, 49, False),   # +5.1 to +8.9
    (64, (32, 8), 5000, 98, True),    # -0.9 to -3.9
    (64, (32, 8), 9000, 17, True),    # -8 to -74: the ordinary launch cuts these rows
    (128, (32, 8), 3000, 33, False),  # +4.5 to +8.8
    (64, (28, 4), 9000, 49, False),   # -2.6 to +10.9
    (64, (28, 4), 9000, 163, True),   # -4.4 to -19.7
    (32, (12, 2), 9000, 133, False),  # -1.2 to +8.0
    (64, (12, 2), 4500, 66, False),   # +5.5 to +8.4
    (128, (12, 2), 9000, 49, False),  # -1.0 to +9.7
    (128, (12, 2), 16000, 162, True), # -5.2 to -20.2
])
def test_decode_steps_share_where_that_is_faster(host_engine, rows, heads, capacity, shared, on):
    e = host_engine(batch=rows, pages=capacity // PAGE + 1, hq=heads[0], hkv=heads[1])
    e._update_sharing({s: list(range(shared)) + [100000 + s] for s in range(rows)})
    assert e._sharing == on


def test_crossing_the_line_keeps_both_captured_steps(host_engine):
    """A batch that fills and drains around it goes back to the step that it had captured; what else changes drops both."""
    e = host_engine()
    sharers = {s: list(range(300)) + [300 + s] for s in range(16)}
    alone = {s: [s] for s in range(16)}
    e._update_sharing(alone)
    assert e._decode_graph is None
    e._decode_graph = "ordinary"
    e._update_sharing(sharers)
    assert e._sharing and e._decode_graph is None
    e._decode_graph = "shared"
    for rows, graph in ((alone, "ordinary"), (sharers, "shared"), (sharers, "shared"), (alone, "ordinary")):
        e._update_sharing(rows)
        assert e._decode_graph == graph
    e._decode_graph = None
    assert e._decode_graph is None
    e._update_sharing(sharers)
    assert e._decode_graph is None


@pytest.mark.parametrize("selective,roles,on", [
    (False, ["plan", "subset"], True),  # every layer attends everything
    (True, ["full", "plan", "subset"], True),
    (True, ["plan", "subset", "subset"], False),
])
def test_decode_steps_without_a_layer_that_shares_are_captured_once(host_engine, selective, roles, on):
    """Planner and subset layers keep their launches: with no other, sharing changes nothing but the captures."""
    e = host_engine()
    e.enable_selective_cache, e.layer_roles = selective, roles
    e._update_sharing({s: list(range(300)) + [300 + s] for s in range(16)})
    assert e._sharing == on
