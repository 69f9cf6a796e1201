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
