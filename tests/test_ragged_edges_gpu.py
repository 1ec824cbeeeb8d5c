"""The ragged operators where an argument or a neighbour is extreme: large caps, rows beside the live ones, windows whose
old pages are gone, far distances, long item lists. Tolerances are ragged_ref's unless a test derives its own."""
import math

import pytest
import torch

from ragged_ref import attend64, attend_check, pages_of
from test_attn_ragged_gpu import fill, verify
from test_rope_gpu import paged

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
ROWS = [1, 1000]  # rows per KV head that max_q announces: one for each kernel


def starts(dev, *counts):
    return torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32, device=dev)


def randn(dev, shape, seed, dtype, gain=1.0):
    return (torch.randn(shape, generator=torch.Generator(device=dev).manual_seed(seed), device=dev) * gain).to(dtype)


# ---------------------------------------------------------------- capped scores
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("slope", [False, True])
@pytest.mark.parametrize("cap", [0.25, 50.0, 1e3, 1e4, 1e6, 1e12, 1e30, 1.9e38])
def test_caps_of_any_size(pkg, dev, dtype, rows, slope, cap):
    """cap tanh(s / cap) is s itself where the cap is large: a fixed cap must not cost the score its digits. fp32 forms it
    with a relative error below 2^-20, so scores below 32 in the base-2 exponent keep to the 1e-4 of attend_check."""
    n, m, D = 5, 300, 128
    q, k, v = randn(dev, (n, 2, D), 1, dtype), randn(dev, (m, 1, D), 2, dtype), randn(dev, (m, 1, D), 3, dtype)
    slopes = torch.tensor([0.05, 0.01], device=dev) if slope else None
    lse = torch.empty((n, 2), device=dev)
    out = pkg.ops.attn_packed(q, k, v, starts(dev, n), starts(dev, m), softcap=cap, slopes=slopes, lse=lse,
                              max_q=rows)
    want, l64, mass = attend64(q, k, v, softcap=cap, slopes=slopes)
    attend_check(out, want, mass, dtype, m, v.abs().max().item())
    assert ((lse.double() - l64).abs() < 2e-4).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("slope", [False, True])
@pytest.mark.parametrize("cap", [1e3, 1e5])
def test_large_cap_beside_scores_beyond_it(pkg, dev, dtype, rows, slope, cap):
    """Some keys score far below -cap (a padded key of the type's lowest values): the others keep their digits."""
    n, m, D = 3, 200, 128
    q, k, v = randn(dev, (n, 2, D), 4, dtype), randn(dev, (m, 1, D), 5, dtype), randn(dev, (m, 1, D), 6, dtype)
    q[..., 0], k[..., 0] = 40.0, 0.0
    k[::17, 0] = 0.0
    k[::17, 0, 0] = -60000.0  # the score -212000
    slopes = torch.tensor([0.05, 0.01], device=dev) if slope else None
    lse = torch.empty((n, 2), device=dev)
    out = pkg.ops.attn_packed(q, k, v, starts(dev, n), starts(dev, m), softcap=cap, slopes=slopes, lse=lse,
                              max_q=rows)
    want, l64, mass = attend64(q, k, v, softcap=cap, slopes=slopes)
    attend_check(out, want, mass, dtype, m, v.abs().max().item())
    assert ((lse.double() - l64).abs() < 2e-4).all()


# ---------------------------------------------------------------- rows beside the live ones
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("opts", [dict(), dict(softcap=20.0), dict(slopes=True), dict(causal=False)])
@pytest.mark.parametrize("heads,D,page", [(4, 128, 64), (4, 64, 16), (3, 64, 64), (4, 128, 24), (4, 128, 4)])
def test_a_sequence_does_not_depend_on_its_neighbours(pkg, dev, rows, opts, heads, D, page):
    """Bit for bit: the first sequence's rows share a tile with rows that hold nothing of its own, and its last page goes on
    behind its end; neither the next sequence's queries nor what stands there may move as much as a rounding."""
    counts, ctx = [33, 40, 1500], [600, 90, 5000]  # the third one's work makes the first one's keys one run
    kc, vc, table, cu, lengths = paged(dev, F16, 1, D, page, counts, ctx, 30)
    fill(kc, vc, table, lengths, 30)
    T = sum(counts)
    q = randn(dev, (T, heads, D), 31, F16, 2.0)
    opts = dict(opts)
    if opts.pop("slopes", False):
        opts["slopes"] = torch.linspace(0.01, 0.3, heads, device=dev)
    got = []
    for gain, junk in ((1.0, 0.0), (30.0, 40.0), (0.0, float("nan"))):
        q2, kc2, vc2 = q.clone(), kc.clone(), vc.clone()
        q2[33:] *= gain
        for b, total in enumerate(lengths.tolist()):
            for c in (kc2, vc2):  # rows behind the end of the last page
                c[table[b, (total - 1) // page].long(), (total - 1) % page + 1:] = junk
        lse = torch.empty((T, heads), device=dev)
        out = pkg.ops.attn_paged(q2, kc2, vc2, table, cu, lengths, lse=lse, max_q=rows, **opts)
        got.append((out[:33].clone(), lse[:33].clone()))
    for out, lse in got[1:]:
        assert torch.equal(out, got[0][0]) and torch.equal(lse, got[0][1])


@pytest.mark.parametrize("rows", ROWS)
def test_a_packed_document_does_not_depend_on_the_next(pkg, dev, rows):
    """The same for packed rows: a tile of keys reaches into the next document."""
    n = [937, 200, 9000]
    q, k, v = (randn(dev, (sum(n), h, 128), s, BF16, 2.0) for h, s in ((2, 33), (1, 34), (1, 35)))
    got = []
    for gain in (1.0, 50.0, float("nan")):
        q2, k2, v2 = q.clone(), k.clone(), v.clone()
        for t in (q2, k2, v2):
            t[937:] *= gain
        cu = starts(dev, *n)
        got.append(pkg.ops.attn_packed(q2, k2, v2, cu, cu, max_q=rows)[:937].clone())
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


# ---------------------------------------------------------------- pages before a window
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("gone", ["no page", "outside", "nan"])
@pytest.mark.parametrize("opts", [dict(window=70), dict(window=300, softcap=20.0), dict(window=33, causal=False, slopes=True)])
@pytest.mark.parametrize("page", [1, 8, 16, 24, 64])
def test_pages_before_the_window_are_not_needed(pkg, dev, dtype, rows, gone, opts, page):
    """A sliding window frees a sequence's old pages: entries without a page, or with one that holds another's values."""
    counts, ctx, H, Hk, D = [1, 40, 150], [700, 330, 900], 4, 2, 64
    kc, vc, table, cu, lengths = paged(dev, dtype, Hk, D, page, counts, ctx, 50)
    fill(kc, vc, table, lengths, 50)
    opts, total = dict(opts), lengths.tolist()
    slopes = torch.linspace(0.01, 0.3, H, device=dev) if opts.pop("slopes", False) else None
    ks = [pages_of(kc, table, b, t).clone() for b, t in enumerate(total)]
    vs = [pages_of(vc, table, b, t).clone() for b, t in enumerate(total)]
    for b, (n, c) in enumerate(zip(counts, ctx)):
        old = max(0, c - opts["window"] + 1) // page  # pages that lie before the first new token's window
        if gone == "nan":
            for cache in (kc, vc):
                cache[table[b, :old].long()] = float("nan")
        else:
            table[b, :old] = -1 if gone == "no page" else kc.shape[0]
    q = randn(dev, (sum(counts), H, D), 51, dtype)
    lse = torch.empty((sum(counts), H), device=dev)
    out = pkg.ops.attn_paged(q, kc, vc, table, cu, lengths, slopes=slopes, lse=lse, max_q=rows, **opts)
    assert pkg._lib.device_status() == 0
    verify(out, lse, q, counts, lambda b: ks[b], lambda b: vs[b], opts, None, dtype, slopes)


# ---------------------------------------------------------------- workspace
@pytest.mark.parametrize("D", [64, 128])
def test_a_workspace_sized_for_tokens_holds_a_chunk(pkg, dev, D):
    n = pkg._lib.load().b2_attn_ragged_workspace_bytes(4, 1, D, 1)
    buf = torch.full((n + (1 << 16),), 85, dtype=torch.uint8, device=dev)
    counts, ctx = [1000, 3, 600], [5000, 700, 20000]
    kc, vc, table, cu, lengths = paged(dev, F16, 1, D, 16, counts, ctx, 60)
    fill(kc, vc, table, lengths, 60)
    q = randn(dev, (sum(counts), 4, D), 61, F16)
    for rows in ROWS:
        want = pkg.ops.attn_paged(q, kc, vc, table, cu, lengths, max_q=rows)
        got = pkg.ops.attn_paged(q, kc, vc, table, cu, lengths, max_q=rows, workspace=buf[:n])
        assert torch.equal(got, want) and (buf[n:] == 85).all()
