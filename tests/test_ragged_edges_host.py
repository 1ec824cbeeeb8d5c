"""What the ragged operators refuse at the ends of their arguments' ranges, without a GPU."""
import ctypes

import pytest

from test_ragged_host import attn, calls  # noqa: F401 (a fixture)

BLOCK = dict(q=4096, sqt=512, sqh=64, out=4096, sot=512, soh=64, lse=0, k=4096, v=4096, s_page=2048, s_row=128, s_head=64,
             table=4096, cu_q=4096, lengths=4096, prefix=0, slopes=0, workspace=4096, table_ld=3, max_pages=3, num_pages=6,
             page_size=16, batch=2, tokens=5, key_rows=6, heads=8, kv_heads=2, dim=64, dtype=0, max_q=1, causal=1, window=0,
             scale=0.125, softcap=0.0)


@pytest.mark.parametrize("kw", [dict(softcap=2.5e38), dict(scale=2.5e38), dict(softcap=1e-40), dict(scale=1e10, softcap=1e-30)])
def test_factors_that_leave_fp32(pkg, calls, kw):
    """log2(e) times scale or softcap, and scale / softcap, must stay finite."""
    with pytest.raises(RuntimeError, match="softcap"):
        pkg.ops.attn_paged(**attn(**kw))
    assert not calls
    block = pkg.ops._RAGGED.pack(*{**BLOCK, **kw}.values())
    assert pkg._lib.load().b2_attn_ragged(block, ctypes.c_void_p(None)) == 1


def test_factors_at_the_ends_are_taken(pkg, calls):
    for kw in (dict(softcap=1.9e38), dict(softcap=1e-30), dict(scale=1e-30)):
        pkg.ops.attn_paged(**attn(**kw))
    assert len(calls) == 3


@pytest.mark.parametrize("dim", [64, 128])
def test_one_workspace_serves_every_call_of_a_dim(pkg, dim):
    """The argument block does not say how large the workspace is: a buffer sized for tokens must hold a chunk's parts too."""
    size = pkg._lib.load().b2_attn_ragged_workspace_bytes
    assert len({size(h, k, dim, n) for h, k in ((8, 2), (32, 8), (7, 1), (5, 5)) for n in (0, 1, 4, 17, 1000, 1 << 30)}) == 1
    assert size(8, 2, dim, 1) > 0 and size(8, 3, dim, 1) == 0 and size(8, 2, 96, 1) == 0
