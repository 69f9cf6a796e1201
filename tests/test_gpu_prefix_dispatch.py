"""Which launch attends a call: the ordinary kernels' bits where they are the faster ones, and the shared kernels right on
either side."""
import pytest
import torch

from delta_amd import kernels as K
from test_gpu_prefix import DEV, Batch, D, i32

pytestmark = pytest.mark.gpu


def exact_tables(b):
    """The batch planned for what it holds."""
    t = dict(b.t, kv_indices=b.t["kv_indices"][:-65].clone())
    b.t = t
    return t, max(len(p) for p in b.pages)


@pytest.mark.parametrize("rows,heads,prefix", [(64, (32, 8), 36), (32, (32, 8), 60), (128, (12, 2), 60), (40, (12, 4), 60)])
def test_decode_that_is_read_as_fast_alone_is_read_alone(rows, heads, prefix):
    """All that the rows may read lies below the line of their (row, kv head) pairs: us shared / ordinary 28.8 / 23.0 (64 rows
    of 8 heads, 64 pages), 20.8 / 15.5 (32 of 8), 25.3 / 16.8 (128 of 2)."""
    b = Batch(*heads, [prefix], [(0, 1 + 7 * i % 50, 1) for i in range(rows)], seed=rows)
    t, most = exact_tables(b)
    got = b.decode(max_pages_per_row=most)
    b.check(got, b.want())
    ws = torch.empty(max(K.decode_workspace_bytes(rows, *heads, most), 256), dtype=torch.uint8, device=DEV)
    want = K.paged_decode(b.q, b.cache, t["kv_indptr"], t["kv_indices"], t["last"], max_pages_per_row=most, workspace=ws)
    assert torch.equal(got[0], want)
    assert K.prefix_attention_workspace_bytes(rows, *heads, most) >= K.decode_workspace_bytes(rows, *heads, most)


@pytest.mark.parametrize("rows,heads,prefix", [(64, (32, 8), 90), (16, (12, 2), 400)])
def test_decode_past_the_line_is_shared(rows, heads, prefix):
    """The bits of the shared launch, whose plan differs by the rows' number alone here; rows longer than planned too."""
    b = Batch(*heads, [prefix], [(0, 1 + 37 * i % 300, 1) for i in range(rows)], seed=rows)
    _, most = exact_tables(b)
    for planned in (most, prefix):
        got = b.decode(max_pages_per_row=planned)
        b.check(got, b.want())
        assert torch.equal(got[0], b.decode(max_pages_per_row=8192)[0])


def test_prompts_of_short_rows_run_on_the_ordinary_launch():
    """Where the caller says how long the rows are; the same results where it does not, and where the rows are longer or out
    only fits the shared launch."""
    b = Batch(32, 8, [18], [(0, 3 + i % 9, 1 + i % 3) for i in range(32)] + [(-1, 30, 20), (-2, 0, 4)], seed=3)
    t, most = exact_tables(b)
    assert most <= 40 and t["kv_indices"].numel() > 64
    want = b.want()
    got = b.prefill(max_pages_per_row=most)
    b.check(got, want)
    ordinary = K.paged_prefill(b.q, b.cache, i32(b.qo), t["kv_indptr"], t["kv_indices"], t["last"], max_qo_len=20)
    assert torch.equal(got[0], ordinary)
    shared = b.prefill()
    b.check(shared, want)
    far = b.prefill(max_pages_per_row=41)
    assert torch.equal(far[0], shared[0]) and torch.equal(far[1], shared[1])
    wide = torch.full((b.q.shape[0], 33 * D + 2), 2.0, dtype=torch.bfloat16, device=DEV)
    o = torch.as_strided(wide, b.q.shape, (33 * D + 2, D, 1), 2)
    assert torch.equal(b.prefill(max_pages_per_row=most, out=o)[0], shared[0])
    assert (wide[:, :2] == 2).all() and (wide[:, 2 + 32 * D:] == 2).all()


@pytest.mark.parametrize("rows,pages", [(1, 32), (1, 33), (3, 21), (4, 16), (5, 13)])
def test_few_pages_in_all_on_either_side_of_the_line(rows, pages):
    b = Batch(12, 2, [pages - 1], [(0, 5 + i, 5) for i in range(rows)], seed=rows)
    exact_tables(b)
    b.check(b.prefill(), b.want())


@pytest.mark.parametrize("hint", [None, 40])
def test_short_prompts_whose_bounds_leave_the_tokens_write_nothing_out_of_place(hint):
    """As on the shared launch: a table that does not fit q ends at its first and last token."""
    b = Batch(12, 2, [9, 4], [(0, 20, 3), (1, 33, 30), (0, 50, 1), (-1, 60, 20)], seed=49)
    t, most = exact_tables(b)
    assert t["kv_indices"].numel() <= 64
    room, lse = torch.full((400, 12, D), 3.0, dtype=torch.bfloat16, device=DEV), torch.full((400, 12), 4.0, device=DEV)
    want = b.want()
    for qo in ([0, 3, 33, 34, 154], [-100, 3, 33, 34, 54], [0, 3, 33, 34, 54]):
        room.fill_(3.0)
        lse.fill_(4.0)
        K.paged_prefill_prefix(b.q, b.cache, i32(qo), t["kv_indptr"], t["kv_indices"], t["last"], t["row_prefix"],
                               t["prefix_indptr"], t["prefix_indices"], max_qo_len=160, max_pages_per_row=hint,
                               out=room[160:214], lse=lse[160:214])
        torch.cuda.synchronize()
        for x, v in ((room, 3), (lse, 4)):
            assert (x[:160] == v).all() and (x[214:] == v).all()
    b.check((room[160:214], lse[160:214]), want)
