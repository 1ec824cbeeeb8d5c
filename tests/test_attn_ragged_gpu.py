"""Attention of packed sequences over a paged cache and over packed rows, against its 64-bit form."""
import pytest
import torch

from ragged_ref import HALF_STEP, attend64, attend_check, pages_of
from test_rope_gpu import paged

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
# Rows per KV head (tokens x group) that max_q announces: one for each kernel.
ROWS = [1, 1000]


def hint(rows, group):
    return -(-rows // group)


def fill(kc, vc, table, lengths, seed):
    """Values in the sequences' rows only: everything else in the caches stays NaN."""
    g = torch.Generator(device=kc.device).manual_seed(seed)
    for b, n in enumerate(lengths.tolist()):
        ps = kc.shape[1]
        j = torch.arange(n, device=kc.device)
        for c in (kc, vc):
            c[table[b, j // ps].long(), j % ps] = torch.randn((n, *c.shape[2:]), generator=g, device=kc.device).to(c.dtype)


def verify(out, lse, q, counts, ks, vs, opts, prefix, dtype, slopes):
    at = 0
    for b, n in enumerate(counts):
        r = slice(at, at + n)
        at += n
        if n == 0:
            continue
        k, v = ks(b), vs(b)
        want, l64, mass = attend64(q[r], k, v, opts.get("scale"), opts.get("causal", True), opts.get("softcap", 0.0),
                                   opts.get("window", 0), slopes, prefix[b] if prefix else 0)
        attend_check(out[r], want, mass, dtype, k.shape[0], v.abs().max().item() if v.numel() else 0.0)
        blind = torch.isinf(l64)
        assert torch.equal(torch.isinf(lse[r]), blind) and (out[r][blind] == 0).all()
        assert ((lse[r].double() - l64)[~blind].abs() < 2e-4).all()


OPTIONS = [dict(), dict(causal=False), dict(window=1), dict(window=70), dict(softcap=5.0), dict(slopes=True),
           dict(prefix=True), dict(scale=0.5, softcap=20.0, window=100, slopes=True, prefix=True),
           dict(causal=False, window=33)]
BATCHES = [  # counts, cached, heads, kv heads, dim, page
    ([1], [0], 4, 1, 128, 16), ([1, 1, 1, 1], [63, 64, 127, 128], 8, 2, 128, 16), ([1] * 9, [0, 1, 5, 700, 15, 16, 17, 300, 2000], 6, 2, 64, 24),
    ([3, 0, 9, 1], [0, 5, 130, 900], 8, 1, 128, 8), ([17, 40], [100, 0], 3, 3, 64, 32), ([130, 1, 65], [60, 1000, 0], 4, 2, 128, 64),
    ([300], [0], 7, 1, 64, 1), ([257], [511], 2, 2, 128, 256)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("batch", range(len(BATCHES)))
@pytest.mark.parametrize("option", range(len(OPTIONS)))
def test_attn_paged(pkg, dev, dtype, batch, option):
    counts, ctx, H, Hk, D, page = BATCHES[batch]
    opts = dict(OPTIONS[option])
    kc, vc, table, cu, lengths = paged(dev, dtype, Hk, D, page, counts, ctx, batch, heads_first=batch % 2 == 1)
    fill(kc, vc, table, lengths, batch)
    T = sum(counts) + 2
    q = (torch.randn((T, H + 1, D), device=dev, generator=torch.Generator(device=dev).manual_seed(7)) * 2).to(dtype)[:, :H]
    slopes = torch.linspace(0.01, 0.5, H, device=dev) if opts.pop("slopes", False) else None
    prefix = None
    if opts.pop("prefix", False):
        prefix = [(n + c) * (b % 3) // 2 for b, (n, c) in enumerate(zip(counts, ctx))]
    out = torch.full((T, H, D), 7.0, dtype=dtype, device=dev)
    lse = torch.full((T, H), 7.0, device=dev)
    pkg.ops.attn_paged(q, kc, vc, table, cu, lengths, slopes=slopes, out=out, lse=lse, max_q=max(counts),
                       prefix=torch.tensor(prefix, dtype=torch.int32, device=dev) if prefix else None, **opts)
    n = sum(counts)
    assert (out[n:] == 7.0).all() and (lse[n:] == 7.0).all()
    total = lengths.tolist()
    verify(out, lse, q, counts, lambda b: pages_of(kc, table, b, total[b]), lambda b: pages_of(vc, table, b, total[b]),
           opts, prefix, dtype, slopes)
    assert pkg._lib.device_status() == 0


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("nq,nk,H,Hk,D", [([5, 200, 1, 0, 33], [5, 200, 1, 0, 33], 4, 2, 128),
                                          ([1, 20, 129], [700, 20, 400], 5, 5, 64), ([4, 3], [0, 2], 8, 1, 128),
                                          ([2, 0], [0, 0], 2, 1, 64)])
def test_attn_packed(pkg, dev, dtype, rows, nq, nk, H, Hk, D):
    """Documents in one buffer, more keys than queries, fewer keys than queries (positions below zero see nothing
    without a prefix), no keys at all."""
    starts = lambda c: torch.tensor([0] + list(torch.tensor(c).cumsum(0)), dtype=torch.int32, device=dev)
    g = torch.Generator(device=dev).manual_seed(sum(nq))
    q = torch.randn((sum(nq), H, D), device=dev, generator=g).to(dtype)
    kv = torch.randn((sum(nk) + 1, 2 * Hk, D), device=dev, generator=g).to(dtype)
    kv[sum(nk):] = float("nan")
    k, v = kv[:sum(nk), :Hk], kv[:sum(nk), Hk:]
    lse = torch.empty((sum(nq), H), device=dev)
    out = pkg.ops.attn_packed(q, k, v, starts(nq), starts(nk), lse=lse, max_q=hint(rows, H // Hk))
    ends = torch.tensor(nk).cumsum(0).tolist()
    verify(out, lse, q, nq, lambda b: k[ends[b] - nk[b]:ends[b]], lambda b: v[ends[b] - nk[b]:ends[b]], {}, None, dtype, None)


@pytest.mark.parametrize("rows", ROWS)
def test_long_context_is_joined_from_parts(pkg, dev, rows):
    """40000 keys for few rows: every item is cut over many CTAs; the same call twice gives the same bits."""
    counts, ctx = [1, 2, 1], [40000, 3, 9000]
    kc, vc, table, cu, lengths = paged(dev, F16, 2, 128, 16, counts, ctx, 5)
    fill(kc, vc, table, lengths, 5)
    q = (torch.randn((4, 8, 128), device=dev) * 3).half()
    lse = torch.empty((4, 8), device=dev)
    out = pkg.ops.attn_paged(q, kc, vc, table, cu, lengths, lse=lse, max_q=hint(rows, 4))
    total = lengths.tolist()
    verify(out, lse, q, counts, lambda b: pages_of(kc, table, b, total[b]), lambda b: pages_of(vc, table, b, total[b]),
           {}, None, F16, None)
    assert torch.equal(out, pkg.ops.attn_paged(q, kc, vc, table, cu, lengths, max_q=hint(rows, 4)))


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("B", [1, 700])
def test_many_short_sequences(pkg, dev, B, rows):
    """More sequences than threads in a CTA, most of them shorter than a unit of keys, some without tokens."""
    counts = [(b * 7) % 3 for b in range(B - 1)] + [2]
    ctx = [(b * 13) % 90 for b in range(B)]
    kc, vc, table, cu, lengths = paged(dev, BF16, 1, 64, 8, counts, ctx, 6)
    fill(kc, vc, table, lengths, 6)
    q = torch.randn((sum(counts), 4, 64), device=dev).to(BF16)
    lse = torch.empty((sum(counts), 4), device=dev)
    out = pkg.ops.attn_paged(q, kc, vc, table, cu, lengths, lse=lse, max_q=hint(rows, 4))
    total = lengths.tolist()
    verify(out, lse, q, counts, lambda b: pages_of(kc, table, b, total[b]), lambda b: pages_of(vc, table, b, total[b]),
           {}, None, BF16, None)


@pytest.mark.parametrize("rows", ROWS)
def test_extreme_scores(pkg, dev, rows):
    """Scores far apart (one key takes all), the types' lowest values among the keys, a cap that saturates."""
    n, m = 3, 200
    q = torch.zeros((n, 2, 64), device=dev).half()
    q[..., 0] = 100.0
    k = torch.zeros((m, 1, 64), device=dev).half()
    k[:, 0, 0] = torch.linspace(-60, 60, m, device=dev)
    k[5, 0, 0] = torch.finfo(F16).min  # the score -6.5e6 * 0.125
    v = torch.randn((m, 1, 64), device=dev).half()
    cu, ck = (torch.tensor([0, x], dtype=torch.int32, device=dev) for x in (n, m))
    for cap in (0.0, 3.0):
        lse = torch.empty((n, 2), device=dev)
        out = pkg.ops.attn_packed(q, k, v, cu, ck, softcap=cap, lse=lse, max_q=hint(rows, 2))
        want, l64, mass = attend64(q, k, v, softcap=cap)
        attend_check(out, want, mass, F16, m, v.abs().max().item())
        assert ((lse.double() - l64).abs() < 2e-4 + 1e-6 * l64.abs()).all()


@pytest.mark.parametrize("rows", ROWS)
def test_bad_pages_are_skipped(pkg, dev, rows):
    kc, vc, table, cu, lengths = paged(dev, F16, 1, 64, 16, [2, 2], [60, 60], 8)
    fill(kc, vc, table, lengths, 8)
    q = torch.randn((4, 2, 64), device=dev).half()
    good = pkg.ops.attn_paged(q, kc, vc, table, cu, lengths, max_q=hint(rows, 2))
    assert pkg._lib.device_status() == 0
    for bad in (-5, kc.shape[0]):
        t2 = table.clone()
        t2[1, 1] = bad
        out = pkg.ops.attn_paged(q, kc, vc, t2, cu, lengths, max_q=hint(rows, 2))
        assert pkg._lib.device_status() == pkg.ops.BAD_PAGE
        assert torch.equal(out[:2], good[:2]) and torch.isfinite(out).all()
    longer = torch.tensor([62, 1 << 30], dtype=torch.int32, device=dev)  # more keys than the table has rows for
    small = table[:, :4].contiguous()
    out = pkg.ops.attn_paged(q, kc, vc, small, cu, longer, max_q=hint(rows, 2))
    assert torch.equal(out[:2], good[:2])
    assert pkg._lib.device_status() == pkg.ops.BAD_PAGE


@pytest.mark.parametrize("rows", ROWS)
def test_graph_replays_with_other_lengths(pkg, dev, rows):
    """Append and attention captured once, replayed as the sequences grow, beside a second graph on another stream."""
    kc, vc, table, cu, lengths = paged(dev, BF16, 2, 128, 16, [1, 1, 1], [300, 20, 150], 9)
    fill(kc, vc, table, lengths, 9)
    inv, _ = pkg.ops.rope_frequencies(128, device=dev)
    qkv = torch.randn((3, 8, 128), device=dev).to(BF16)
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]

    def step():
        qr = pkg.ops.kv_append(k, v, kc, vc, table, cu, lengths, inv_freq=inv, q=q)
        return qr, pkg.ops.attn_paged(qr, kc, vc, table, cu, lengths, max_q=hint(rows, 2))

    step()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = step()
        graphs.append((g, r))
    for at in ([10, 3, 160], [301, 21, 151], [64, 16, 1]):
        lengths.copy_(torch.tensor(at, dtype=torch.int32))
        qkv.normal_()
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        qr, want = step()
        for _, (gq, got) in graphs:
            # bits: a length of 160 reads rows of the third sequence that were never written, which are NaN
            assert torch.equal(gq, qr) and torch.equal(got.view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_prompt_in_chunks_then_tokens(pkg, dev, dtype):
    """The operators as a decoder uses them: two prompts read in ragged chunks, then tokens one by one, against one
    64-bit pass over the whole sequences."""
    from ragged_ref import rope64
    H, Hk, D, page = 8, 2, 128, 16
    total = [150, 70]
    chunks = [[100, 3], [49, 66], [1, 1]]
    kc, vc, table, _, _ = paged(dev, dtype, Hk, D, page, [0, 0], total, 11)
    inv, _ = pkg.ops.rope_frequencies(D, device=dev)
    data = [torch.randn((n, H + 2 * Hk, D), device=dev).to(dtype) for n in total]
    done = [0, 0]
    got = [[], []]
    for step in chunks:
        x = torch.cat([data[b][done[b]:done[b] + n] for b, n in enumerate(step)])
        done = [d + n for d, n in zip(done, step)]
        cu = torch.tensor([0, step[0], sum(step)], dtype=torch.int32, device=dev)
        lengths = torch.tensor(done, dtype=torch.int32, device=dev)
        q = pkg.ops.kv_append(x[:, H:H + Hk], x[:, H + Hk:], kc, vc, table, cu, lengths, inv_freq=inv, q=x[:, :H])
        out = pkg.ops.attn_paged(q, kc, vc, table, cu, lengths)
        got[0].append(out[:step[0]])
        got[1].append(out[step[0]:])
    for b, n in enumerate(total):
        pos = torch.arange(n, device=dev)
        x = data[b]
        # the cache and the rotated queries hold 16-bit values: half a step each in q and k moves a score by
        # at most |q||k| scale * step, which the comparison takes from the rounded values instead
        q = rope64(x[:, :H], pos, inv).to(dtype)
        k = rope64(x[:, H:H + Hk], pos, inv).to(dtype)
        want, _, mass = attend64(q, k, x[:, H + Hk:])
        have = torch.cat(got[b])
        # a value that the kernel's fp32 rounds the other way moves q or k by a whole step: scores by 2 half-steps
        # sum |q k| scale, below 4 |q|.|k| scale half-steps in the weight
        mag = (q.double().abs().amax() * 0 + x[:, :H].double().pow(2).sum(-1).sqrt().max()
               * x[:, H:H + Hk].double().pow(2).sum(-1).sqrt().max() * D ** -0.5)
        rare = 4 * HALF_STEP[dtype] * 0.02 * mag  # at most 1 value in 50 lies that close to a border
        err = (have.double() - want).abs()
        tol = HALF_STEP[dtype] * want.abs() + (2 * HALF_STEP[dtype] + 4e-4 + rare) * mass + 2.0 ** -24 * n
        assert (err <= tol).all(), (err - tol).max()


def test_other_stream_and_workspace(pkg, dev):
    kc, vc, table, cu, lengths = paged(dev, F16, 2, 64, 16, [1], [2000], 12)
    fill(kc, vc, table, lengths, 12)
    q = torch.randn((1, 4, 64), device=dev).half()
    want = pkg.ops.attn_paged(q, kc, vc, table, cu, lengths)
    ws = torch.empty(64 << 20, dtype=torch.uint8, device=dev)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = pkg.ops.attn_paged(q, kc, vc, table, cu, lengths, workspace=ws)
    s.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("rows", ROWS)
def test_sequences_share_pages(pkg, dev, rows):
    """Two sequences whose tables begin with the same pages (a common prompt), the second one longer."""
    kc, vc, table, _, _ = paged(dev, F16, 2, 128, 16, [0, 0], [64, 100], 13)
    table[1, :4] = table[0, :4]
    lengths = torch.tensor([64, 100], dtype=torch.int32, device=dev)
    fill(kc, vc, table, lengths, 13)
    q = torch.randn((5, 8, 128), device=dev).half()
    cu = torch.tensor([0, 2, 5], dtype=torch.int32, device=dev)
    lse = torch.empty((5, 8), device=dev)
    out = pkg.ops.attn_paged(q, kc, vc, table, cu, lengths, lse=lse, max_q=hint(rows, 4))
    total = [64, 100]
    verify(out, lse, q, [2, 3], lambda b: pages_of(kc, table, b, total[b]), lambda b: pages_of(vc, table, b, total[b]), {},
           None, F16, None)


@pytest.mark.parametrize("rows", ROWS)
def test_cache_offsets_past_32_bits(pkg, dev, rows):
    """Pages 1.5 * 2^30 elements apart (9.7 GB in all): append, rotation and attention reach them."""
    step, page, Hk, D = 3 << 29, 16, 1, 64
    buf = torch.empty(3 * step, dtype=F16, device=dev)
    cache = lambda at: buf[at:].as_strided((3, page, Hk, D), (step, D, D, 1))
    kc, vc = cache(0), cache(1 << 20)
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=dev)
    n = 40
    x = torch.randn((n, 4, D), device=dev).half()
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    lengths = torch.tensor([n], dtype=torch.int32, device=dev)
    pkg.ops.kv_append(x[:, 2:3], x[:, 3:], kc, vc, table, cu, lengths)
    assert torch.equal(pages_of(kc, table, 0, n), x[:, 2:3]) and torch.equal(pages_of(vc, table, 0, n), x[:, 3:])
    lse = torch.empty((n, 2), device=dev)
    out = pkg.ops.attn_paged(x[:, :2], kc, vc, table, cu, lengths, lse=lse, max_q=hint(rows, 2))
    verify(out, lse, x[:, :2], [n], lambda b: x[:, 2:3], lambda b: x[:, 3:], {}, None, F16, None)


@pytest.mark.parametrize("rows", ROWS)
def test_calls_that_overlap(pkg, dev, rows):
    """Calls on several streams at once, each with its own workspace, give what they give alone."""
    data = []
    for i in range(4):
        kc, vc, table, cu, lengths = paged(dev, F16, 2, 64, 16, [3, 1], [3000 + 100 * i, 50], 20 + i)
        fill(kc, vc, table, lengths, 20 + i)
        data.append((torch.randn((4, 4, 64), device=dev).half(), kc, vc, table, cu, lengths))
    alone = [pkg.ops.attn_paged(*d, max_q=hint(rows, 2)) for d in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in data]
    for _ in range(3):
        got = []
        for s, d in zip(streams, data):
            with torch.cuda.stream(s):
                got.append(pkg.ops.attn_paged(*d, max_q=hint(rows, 2)))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(alone, got))


def test_bound_of_the_cap_on_both_paths(pkg, dev):
    """Scores across the whole of tanh, small ones beside large ones, so that both ways of computing the cap are taken."""
    n = 130
    q = torch.randn((n, 2, 128), device=dev).half()
    k = torch.randn((400, 1, 128), device=dev).half()
    k[200:] *= 20
    v = torch.randn((400, 1, 128), device=dev).half()
    cu, ck = (torch.tensor([0, x], dtype=torch.int32, device=dev) for x in (n, 400))
    for cap in (0.5, 8.0, 40.0):
        for slopes in (None, torch.tensor([0.1, 0.02], device=dev)):
            out = pkg.ops.attn_packed(q, k, v, cu, ck, softcap=cap, slopes=slopes, max_q=1000)
            want, _, mass = attend64(q, k, v, softcap=cap, slopes=slopes)
            attend_check(out, want, mass, F16, 400, v.abs().max().item())


def test_single_elements_have_no_stride(pkg, dev):
    """One token, one head, one page of one row: torch's strides of such dimensions mean nothing and may be odd."""
    buf = torch.randn(4096, device=dev).half()
    q = buf[:64].as_strided((1, 1, 64), (513, 7, 1))
    kc = buf[64:128].as_strided((1, 1, 1, 64), (33, 5, 3, 1))
    vc = buf[128:192].as_strided((1, 1, 1, 64), (9, 11, 13, 1))
    table = torch.zeros((1, 1), dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 1], dtype=torch.int32, device=dev)
    one = torch.ones(1, dtype=torch.int32, device=dev)
    for rows in ROWS:
        assert torch.equal(pkg.ops.attn_paged(q, kc, vc, table, cu, one, max_q=rows)[0, 0], vc[0, 0, 0])
    inv, _ = pkg.ops.rope_frequencies(64, device=dev)
    pkg.ops.kv_append(q, q, kc, vc, table, cu, one, inv_freq=inv)
    assert torch.equal(vc[0, 0, 0], q[0, 0]) and torch.equal(kc[0, 0, 0], q[0, 0])  # position 0 does not turn
