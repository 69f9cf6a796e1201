"""What the engine's steps over shared pages attend, against 64-bit softmax over each request's own pages: prompt steps of
sharers alone and beside a long prompt, captured decode steps that go from one launch to the other and back; and forked
sequences against caches of their own.  Tolerances as in test_gpu_prefix.py (its bound on sum |q_i k_i| is asserted)."""
import pytest
import torch

import delta_amd.backend as backend
import delta_amd.kernels as K
from test_gpu_engine import make_engine
from test_gpu_prefix import DEV, PAGE, Batch, D, _caches, i32, indptr
from test_gpu_prefix_engine import check_decode_layer, prompt

pytestmark = pytest.mark.gpu


def rows_of(cache, q, pages, kv_len, qn):
    """A ``Batch`` of given rows: its ``want`` and ``check``."""
    b = Batch.__new__(Batch)
    b.cache, b.q, b.pages, b.kv_len, b.qo, b.hq, b.hkv = cache, q, pages, kv_len, indptr(qn), q.shape[1], cache.shape[3]
    return b


def check_prompts(eng, monkeypatch):
    """Checks every shared prompt launch of two layers; returns the (new tokens, prefix) of their rows, step by step."""
    steps, first, last = [], eng.model.layers[0], eng.model.layers[-1]
    launch = K.paged_prefill_prefix

    def checked(q, cache, *tables, **kw):
        lse = torch.empty(q.shape[:2], device=q.device)
        o = launch(q, cache, *tables, lse=lse, **kw)
        if cache.data_ptr() not in [l.attention.kv_cache.kv_cache.data_ptr() for l in (first, last)]:
            return o
        reqs = [eng.scheduler.request_in(s) for s in eng.scheduler.occupied()]
        qn = [len(r.next_input()) for r in reqs]
        if cache.data_ptr() == first.attention.kv_cache.kv_cache.data_ptr():
            steps.append(list(zip(qn, tables[4].tolist())))
        b = rows_of(cache, q, [r.pages for r in reqs], [r.kv_len() for r in reqs], qn)
        used = cache[torch.tensor(sorted({p for r in reqs for p in r.pages}), device=cache.device)]
        assert q.float().norm(dim=-1).max() * used[:, 0].float().norm(dim=-1).max() / D ** 0.5 <= 12
        b.check((o, lse), b.want())
        return o

    monkeypatch.setattr(K, "paged_prefill_prefix", checked)
    return steps


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_shared_prompt_steps_attend_each_requests_own_pages(dtype, monkeypatch):
    """Sixteen prompts of one prefix with parts of their own, four more that come while others decode, and forks."""
    eng = make_engine(B=16, max_len=5376, dtype=dtype)
    steps = check_prompts(eng, monkeypatch)
    eng.add_requests([prompt(1 + 7 * i, i) for i in range(20)], [4800 + 160 + i for i in range(20)], [],
                     prefix_ids=prompt(4805, 0))

    def on_step(e, i):
        r = e.scheduler.requests[19]
        if len(r.generated) == 3 and e.scheduler.free_slot() is not None:
            e.fork_request(19, prompt(9, 50), max_length=4800 + 190)

    eng.run_scheduler_loop(on_step=on_step)
    assert eng.page_pool.available == eng.page_pool.total_pages
    assert [q for q, _ in steps[0]] == [6 + 7 * i for i in range(16)] and len(steps) >= 3
    assert any(q == 1 for s in steps for q, _ in s) and all(max(p for _, p in s) == 0 for s in steps)


def test_a_long_prompt_beside_sharers(monkeypatch):
    """A row past SHARING_PAIRS, which has no prefix, in the sharers' launch; and the ordinary launch where that is faster."""
    for longest, shared in ((600, True), (5000, False)):
        eng = make_engine(B=16, max_len=5376)
        group = eng.model.config.n_head // eng.model.config.n_local_heads
        steps = check_prompts(eng, monkeypatch)
        eng.add_requests([prompt(2 + i, i) for i in range(15)], 4800 + 60, [], prefix_ids=prompt(4800, 0))
        if shared:
            assert longest * group > backend.SHARING_PAIRS

        def on_step(e, i):
            if i == 1:
                e.add_requests([prompt(longest, 99)], longest + 4, [])

        ordinary = []
        launch = K.paged_prefill
        monkeypatch.setattr(K, "paged_prefill", lambda *a, **kw: ordinary.append(kw["max_qo_len"]) or launch(*a, **kw))
        if not shared:  # (on this small shape a long prompt alone does not make the ordinary launch the faster one)
            monkeypatch.setattr(backend, "prompt_step_us", lambda qo, *a: (1.0, 0.0) if max(qo) > 1000 else (0.0, 1.0))
        eng.run_scheduler_loop(on_step=on_step)
        mixed = [s for s in steps if any(q == longest for q, _ in s)]
        if shared:
            (rows,) = mixed
            assert [p for q, p in rows] == [-1 if q == longest else 0 for q, _ in rows] and longest not in ordinary
        else:
            assert not mixed and longest in ordinary and len(steps) == 1
        assert eng.page_pool.available == eng.page_pool.total_pages
        monkeypatch.undo()


def test_sharing_goes_off_and_on_in_one_loop():
    """Rows that end take the batch below the line (15 rows of 280 common pages on 2 kv heads spare 7840 page-heads), forks
    bring it back: every replayed step's attention is the oracle's, on two captured steps in all."""
    eng = make_engine(B=16, max_len=5120, graph=True)
    layer = eng.model.layers[0]
    capture, static = eng._capture_decode_graph, {}

    def recorded():  # the clones that the captured step writes at every replay
        layer.attention.record = []
        capture()
        static[eng._sharing] = layer.attention.record[-1]
        layer.attention.record = None

    eng._capture_decode_graph = recorded
    caps = [4480 + 200] * 16
    caps[3] = 4480 + 14
    eng.add_requests([prompt(2 + i % 5, i) for i in range(16)], caps, [], prefix_ids=prompt(4480, 0))
    state, checked, crossings = [None], {True: 0, False: 0}, [0]

    def on_step(e, i):
        replays = e._decode_graph_stats["replays"]
        if replays != state[0] and state[0] is not None:
            live = {s: e.scheduler.request_in(s) for s in e.scheduler.occupied()}
            if checked[e._sharing] % 3 == 0:
                layer.attention.record = [static[e._sharing]]
                rows = {s: (r.pages, r.kv_len()) for s, r in list(live.items())[i % 4::4] if not r.finished}
                check_decode_layer(layer, rows, f"step {i} sharing {e._sharing}")
                layer.attention.record = None
            checked[e._sharing] += 1
        state[0] = replays
        if not e._sharing and i % 4 == 0 and crossings[0] < 4 and e.scheduler.free_slot() is not None:
            e.fork_request(1, prompt(3, i), max_length=len(e.scheduler.requests[1].prompt) + len(e.scheduler.requests[1].generated) + 11)
            assert e._sharing
            crossings[0] += 1

    eng.run_scheduler_loop(on_step=on_step)
    assert crossings[0] == 4 and min(checked.values()) >= 12
    assert eng._decode_graph_stats["captures"] == 2 and eng._decode_graph_failed is None and not eng._sharing
    assert eng.page_pool.available == eng.page_pool.total_pages


def test_forked_sequences_attend_what_caches_of_their_own_hold():
    """A sequence of 150 tokens forks three ways: nine full pages shared, the tenth (6 tokens) copied, a prompt and a decode
    step appended to each branch; against caches in which every branch's whole context was written by itself."""
    hq, hkv, n0, L = 12, 2, 150, 3
    caches = _caches(L, 80, hkv, torch.bfloat16, seed=31)
    branches, g = [5, 23, 17], torch.Generator(device=DEV).manual_seed(32)
    own = [[20 + 5 * i + k for k in range(3)] for i in range(3)]
    alone = [torch.zeros(36, 2, PAGE, hkv, D, dtype=torch.bfloat16, device=DEV) for _ in range(L)]  # 12 pages a branch
    for a, c in zip(alone, caches):
        for i in range(3):
            a[12 * i:12 * i + 9] = c[:9]
            a[12 * i + 9, :, :n0 % PAGE] = c[9, :, :n0 % PAGE]
    K.copy_pages(caches, i32([9] * 3), i32([o[0] for o in own]), tokens=i32([n0 % PAGE] * 3))
    lens = [n0] * 3
    for new in (branches, [1, 1, 1]):
        at, lens = lens, [n + k for n, k in zip(lens, new)]
        npg = [-(-n // PAGE) for n in lens]
        rows = [list(range(9)) + o[:c - 9] for o, c in zip(own, npg)]
        ap, ip, ind = i32(indptr(new)), i32(indptr(npg)), i32([p for r in rows for p in r] + [-1] * 65)
        last, px = i32([(n - 1) % PAGE + 1 for n in lens]), (i32([0, 0, 0]), i32([0, 9]), i32(list(range(9))))
        for cache, a in zip(caches, alone):
            k, v, q = (torch.randn(sum(new), h, D, device=DEV, generator=g).to(torch.bfloat16) for h in (hkv, hkv, hq))
            K.append_kv(k, v, ap, cache, ind, ip, last)
            t = 0
            for i in range(3):
                for pos in range(at[i], lens[i]):
                    a[12 * i + pos // PAGE, 0, pos % PAGE], a[12 * i + pos // PAGE, 1, pos % PAGE] = k[t], v[t]
                    t += 1
            lse = torch.empty(sum(new), hq, device=DEV)
            if new is branches:
                o = K.paged_prefill_prefix(q, cache, ap, ip, ind, last, *px, max_qo_len=max(new), lse=lse)
            else:
                o = K.paged_decode_prefix(q, cache, ip, ind, last, *px, max_pages_per_row=4096, lse=lse)
            b = rows_of(a, q, [list(range(12 * i, 12 * i + c)) for i, c in enumerate(npg)], lens, new)
            b.check((o, lse), b.want())
    for c, a in zip(caches, alone):
        for i, o in enumerate(own):
            assert torch.equal(c[o[0], :, :n0 % PAGE], a[12 * i + 9, :, :n0 % PAGE])
            assert torch.equal(c[9, :, :n0 % PAGE], a[12 * i + 9, :, :n0 % PAGE])
