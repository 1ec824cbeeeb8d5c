"""The ragged operators where an argument or a neighbour is extreme: large caps, rows beside the live ones, windows whose
old pages are gone, far distances, long item lists. Tolerances are ragged_ref's unless a test derives its own."""
import math

import pytest
import torch

from ragged_ref import HALF_STEP, attend64, attend_check, check, pages_of, rope64, rope_bound
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


# ---------------------------------------------------------------- bias of far keys
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("cap", [0.0, 9.0])
@pytest.mark.parametrize("slope", [0.37, 0.0507, -0.2113])
def test_bias_where_every_key_is_far(pkg, dev, dtype, rows, cap, slope):
    """More queries than keys (the first query is 20000 positions before the keys' middle) and a bias that grows with the distance:
    all weights are differences of large biases. A score of magnitude B in the base-2 exponent, formed in fp32 from
    product and sum, is off by 2 * 2^-24 B, a weight by ln 2 times that, and the sum by as much."""
    n, m, H, D = 20000, 96, 2, 128
    q, k, v = randn(dev, (n, H, D), 40, dtype), randn(dev, (m, 1, D), 41, dtype), randn(dev, (m, 1, D), 42, dtype)
    slopes = torch.tensor([slope, slope / 3], device=dev)
    lse = torch.empty((n, H), device=dev)
    out = pkg.ops.attn_packed(q, k, v, starts(dev, n), starts(dev, m), causal=False, softcap=cap, slopes=slopes, lse=lse, max_q=rows)
    r = torch.arange(0, n, 97, device=dev)
    dist = (r[:, None] + (m - n) - torch.arange(m, device=dev)[None, :]).abs().double()
    for h in range(H):
        s = q[r, h].double() @ k[:, 0].double().t() * D ** -0.5
        if cap:
            s = cap * torch.tanh(s / cap)
        s = s - slopes[h].double() * dist
        w = torch.softmax(s, 1)
        want, mass = w @ v[:, 0].double(), w @ v[:, 0].double().abs()
        B = s.abs().amax(1, keepdim=True) / math.log(2)
        extra = (HALF_STEP[dtype] + 4e-4 + 2 * math.log(2) * 2.0 ** -23 * B) * mass
        if dtype == F16:
            extra = extra + m * 2.0 ** -25 * v.abs().max().item()
        check(out[r, h], want, extra, dtype)
        assert ((lse[r, h].double() - torch.logsumexp(s, 1)).abs() < 2e-4 + 2.0 ** -22 * B[:, 0]).all()


# ---------------------------------------------------------------- paths that take a special shape
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,page,opts", [(64, 16, {}), (128, 16, dict(softcap=10.0)), (64, 3, {}), (128, 64, dict(window=20))])
def test_more_items_than_a_list_holds(pkg, dev, dtype, D, page, opts):
    """1700 short sequences of 8 KV heads are about 70 items per CTA of the 256-row kernel, which describes 48 at a time; some of
    several units among them. Compared with one padded 64-bit computation."""
    B, Hk, G = 1700, 8, 2
    counts = [(7 * b) % 4 for b in range(B)]
    ctx = [(37 * b) % 60 + (300 if b % 50 == 0 else 0) for b in range(B)]
    kc, vc, table, cu, lengths = paged(dev, dtype, Hk, D, page, counts, ctx, 70)
    m = max(n + c for n, c in zip(counts, ctx))
    j = torch.arange(m, device=dev)[None, :]
    there = j < lengths[:, None]
    at = table[:, :-(-m // page)].long().repeat_interleave(page, 1)[:, :m].masked_fill(~there, 0)
    k, v = (randn(dev, (B, m, Hk, D), s, dtype) for s in (71, 72))
    row = (j % page).expand(B, m)
    for cache, x in ((kc, k), (vc, v)):
        cache[at[there], row[there]] = x[there]
    seq = torch.repeat_interleave(torch.arange(B, device=dev), cu.diff().long())
    pos = torch.arange(len(seq), device=dev) - cu[seq + 1].long() + lengths[seq].long()
    q = randn(dev, (len(seq), Hk * G, D), 73, dtype)
    lse = torch.empty((len(seq), Hk * G), device=dev)
    out = pkg.ops.attn_paged(q, kc, vc, table, cu, lengths, lse=lse, max_q=1000, **opts)
    assert pkg._lib.device_status() == 0
    vis = (j <= pos[:, None]) & (pos[:, None] - j < opts.get("window", 1 << 30))
    vmax = v.abs().max().item()
    for h in range(Hk * G):
        s = torch.einsum("td,tmd->tm", q[:, h].double(), k[seq, :, h // G].double()) * D ** -0.5
        if "softcap" in opts:
            s = opts["softcap"] * torch.tanh(s / opts["softcap"])
        s = s.masked_fill(~vis, -math.inf)
        w, vv = torch.softmax(s, 1), v[seq, :, h // G].double()
        attend_check(out[:, h], torch.einsum("tm,tmd->td", w, vv), torch.einsum("tm,tmd->td", w, vv.abs()), dtype, m, vmax)
        assert ((lse[:, h].double() - torch.logsumexp(s, 1)).abs() < 2e-4).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("page", [16, 24, 128])
@pytest.mark.parametrize("H,Hk,D", [(6, 2, 64), (12, 4, 128), (5, 1, 64)])
@pytest.mark.parametrize("opts", [dict(), dict(softcap=5.0), dict(slopes=True, window=90), dict(causal=False)])
def test_groups_that_no_box_of_queries_holds(pkg, dev, dtype, page, H, Hk, D, opts):
    """Three or five heads per KV head do not divide a tile's 128 rows: keys come by TMA, queries row by row."""
    counts, ctx = [100, 2, 43], [50, 300, 0]
    kc, vc, table, cu, lengths = paged(dev, dtype, Hk, D, page, counts, ctx, 80)
    fill(kc, vc, table, lengths, 80)
    q = randn(dev, (sum(counts), H, D), 81, dtype, 2.0)
    opts, total = dict(opts), lengths.tolist()
    slopes = torch.linspace(0.01, 0.3, H, device=dev) if opts.pop("slopes", False) else None
    lse = torch.empty((sum(counts), H), device=dev)
    out = pkg.ops.attn_paged(q, kc, vc, table, cu, lengths, slopes=slopes, lse=lse, max_q=100, **opts)
    verify(out, lse, q, counts, lambda b: pages_of(kc, table, b, total[b]), lambda b: pages_of(vc, table, b, total[b]),
           opts, None, dtype, slopes)


@pytest.mark.parametrize("H,D", [(32, 64), (64, 128), (128, 128), (160, 64), (300, 64)])
@pytest.mark.parametrize("opts", [dict(), dict(softcap=5.0, slopes=True, window=90)])
def test_many_heads_on_one_kv_head(pkg, dev, H, D, opts):
    """A token of 128 heads is a tile by itself; one of 160 or 300 begins and ends inside tiles."""
    counts, ctx = [3, 1, 2], [140, 300, 0]
    kc, vc, table, cu, lengths = paged(dev, BF16, 1, D, 16, counts, ctx, 85)
    fill(kc, vc, table, lengths, 85)
    q = randn(dev, (sum(counts), H, D), 86, BF16, 2.0)
    opts, total = dict(opts), lengths.tolist()
    slopes = torch.linspace(0.01, 0.3, H, device=dev) if opts.pop("slopes", False) else None
    lse = torch.empty((sum(counts), H), device=dev)
    out = pkg.ops.attn_paged(q, kc, vc, table, cu, lengths, slopes=slopes, lse=lse, **opts)
    verify(out, lse, q, counts, lambda b: pages_of(kc, table, b, total[b]), lambda b: pages_of(vc, table, b, total[b]),
           opts, None, BF16, slopes)


@pytest.mark.parametrize("dtype", [F16, BF16, torch.float32])
@pytest.mark.parametrize("tokens", [592, 593, 594, 595, 1777])
@pytest.mark.parametrize("dim,rot,interleaved", [(64, 64, False), (96, 32, True), (10, 6, False)])
def test_four_tokens_per_cta_and_the_rest(pkg, dev, dtype, tokens, dim, rot, interleaved):
    """Many tokens are rotated four to a CTA: counts that leave one, two or three in the last one, each token with its own
    angles and its own place in the cache; heads of 10 values go value by value."""
    inv, _ = pkg.ops.rope_frequencies(rot, device=dev)
    x = randn(dev, (tokens, 3, dim), 90, dtype)
    pos = torch.randint(0, 1 << 20, (tokens,), generator=torch.Generator().manual_seed(tokens)).to(dev)
    want = rope64(x, pos, inv, interleaved)
    check(pkg.ops.rope(x, pos, inv, interleaved=interleaved), want, rope_bound(x, want, inv, interleaved), dtype)
    counts = [tokens - 5 - tokens // 3 - 2, 5, 0, tokens // 3]  # two rows behind the last sequence
    ctx = [30, 0, 9, 100]
    kc, vc, table, cu, lengths = paged(dev, dtype, 1, dim, 16, counts, ctx, 91)
    q, k, v = x[:, :1], x[:, 1:2], x[:, 2:]
    q_out = torch.full((tokens, 1, dim), 7.0, dtype=dtype, device=dev)
    pkg.ops.kv_append(k, v, kc, vc, table, cu, lengths, inv_freq=inv, q=q, q_out=q_out, interleaved=interleaved)
    assert (q_out[-2:] == 7.0).all() and pkg._lib.device_status() == 0
    at = 0
    for b, (n, c) in enumerate(zip(counts, ctx)):
        r, here = slice(at, at + n), torch.arange(c, c + n, device=dev)
        at += n
        for got, src in ((q_out[r], q[r]), (pages_of(kc, table, b, c + n)[c:], k[r])):
            want = rope64(src, here, inv, interleaved)
            check(got, want, rope_bound(src, want, inv, interleaved), dtype)
        assert torch.equal(pages_of(vc, table, b, c + n)[c:], v[r])


# ---------------------------------------------------------------- weights of single tokens
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("keys", [7, 60, 900])
def test_few_rows_are_off_by_their_rounding(pkg, dev, dtype, D, keys):
    """The kernel for few rows keeps its weights to 16 bits or more, so the error of its output is the rounding of the output
    to the type. Beside that, in the mean square: scores and exponentials in fp32 (1e-6) and weights to 2^-16 (bf16) or
    2^-22 (fp16), at most 2e-5 against 2^-9.3 or 2^-12.3: less than a thousandth of the error. 2 % is allowed."""
    B = 40
    counts, ctx = [1] * B, [keys - 1] * B
    kc, vc, table, cu, lengths = paged(dev, dtype, 2, D, 16, counts, ctx, 95)
    fill(kc, vc, table, lengths, 95)
    q = randn(dev, (B, 8, D), 96, dtype, 2.0)
    out = pkg.ops.attn_paged(q, kc, vc, table, cu, lengths)
    want = torch.cat([attend64(q[b:b + 1], pages_of(kc, table, b, keys), pages_of(vc, table, b, keys))[0] for b in range(B)])
    assert (out.double() - want).norm() < 1.02 * (want.to(dtype).double() - want).norm()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("D", [64, 128])
def test_infinite_values_of_visible_keys(pkg, dev, dtype, rows, D):
    """An infinity in v comes out as itself where its key has weight (at least 2^-9 here), and touches its column only."""
    m = 24
    q, k, v = randn(dev, (1, 2, D), 97, dtype, 0.5), randn(dev, (m, 1, D), 98, dtype, 0.5), randn(dev, (m, 1, D), 99, dtype)
    clean = v.clone()
    v[3, 0, 5], v[7, 0, 9], v[0, 0, D - 1] = math.inf, -math.inf, math.inf
    v[2, 0, 11] = torch.finfo(dtype).max
    out = pkg.ops.attn_packed(q, k, v, starts(dev, 1), starts(dev, m), max_q=rows)
    assert (out[0, :, 5] == math.inf).all() and (out[0, :, 9] == -math.inf).all() and (out[0, :, D - 1] == math.inf).all()
    rest = [c for c in range(D) if c not in (5, 9, 11, D - 1)]
    want, _, mass = attend64(q, k, clean)
    attend_check(out[..., rest], want[..., rest], mass[..., rest], dtype, m, clean.abs().max().item())
    assert torch.isfinite(out[..., 11]).all()
