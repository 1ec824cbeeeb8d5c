"""Rotary positions and the append to a paged cache on the GPU, against their 64-bit forms."""
import pytest
import torch

from ragged_ref import check, pages_of, rope64, rope_bound

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def freqs(pkg, rot, dev, **kw):
    return pkg.ops.rope_frequencies(rot, device=dev, **kw) if rot else (torch.empty(0, device=dev), 1.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,rot", [(1, 1, 64, 64), (5, 3, 128, 128), (33, 2, 96, 32), (7, 20, 256, 64),
                                                  (4, 2, 10, 6), (3, 5, 2, 2), (2, 1, 80, 40), (9, 4, 128, 0),
                                                  (600, 8, 128, 128), (2, 3, 1024, 1024)])
def test_rope(pkg, dev, dtype, interleaved, tokens, heads, dim, rot):
    g = torch.Generator().manual_seed(tokens * dim)
    x = torch.randn((tokens, heads, dim), generator=g).to(dtype).to(dev)
    pos = torch.randint(0, 1 << 20, (tokens,), generator=g).to(dev)
    inv, ms = freqs(pkg, rot, dev, base=500000.0)
    got = pkg.ops.rope(x, pos, inv, interleaved=interleaved)
    want = rope64(x, pos, inv, interleaved)
    check(got, want, rope_bound(x, want, inv, interleaved), dtype)
    assert torch.equal(got[..., rot:], x[..., rot:])


def test_rope_far_negative_and_strided(pkg, dev):
    """Positions up to 2^31, negative ones (they undo the rotation), views of one buffer, in place, mscale."""
    inv, ms = pkg.ops.rope_frequencies(128, base=1e6, scaling="ramp", factor=16.0, original_length=4096, device=dev)
    assert abs(ms - 1.27725887) < 1e-6
    buf = torch.randn((40, 12, 128), device=dev)
    x = buf[::2, 3:8]
    pos = torch.linspace(0, 2 ** 31 - 1, 20, dtype=torch.float64).long().to(dev)
    want = rope64(x, pos, inv, False, ms)
    keep = buf.clone()
    out = pkg.ops.rope(x, pos, inv, mscale=ms, out=x)
    assert out.data_ptr() == x.data_ptr()
    # the 64-bit form itself rounds its angle: 2^31 * 2^-53
    check(x, want, rope_bound(keep[::2, 3:8], want, inv, False, ms) + 2.0 ** -20, torch.float32)
    back = pkg.ops.rope(x, -pos, inv, mscale=1 / ms)
    assert (back - keep[::2, 3:8]).abs().max() < 4e-6 * keep.abs().max()
    other = torch.ones_like(buf, dtype=torch.bool)
    other[::2, 3:8] = False
    assert torch.equal(buf[other], keep[other])
    # rows that do not start on 16 bytes take the value-by-value path
    odd = torch.randn((6, 2, 131), device=dev).half()[..., 1:129]
    p6 = torch.arange(6, device=dev)
    want = rope64(odd, p6, inv)
    check(pkg.ops.rope(odd, p6, inv), want, rope_bound(odd, want, inv), torch.float16)


def test_rope_gradient_is_the_turn_back(pkg, dev):
    """d(out . w)/dx = rope(w, -positions), against differences of the 64-bit form."""
    inv, _ = pkg.ops.rope_frequencies(8, device=dev)
    x, w = torch.randn((5, 2, 8), device=dev), torch.randn((5, 2, 8), device=dev)
    pos = torch.arange(5, device=dev) * 37
    grad = pkg.ops.rope(w, -pos, inv)
    for e in range(8):
        d = torch.zeros_like(x)
        d[..., e] = 1
        diff = ((rope64(x + d, pos, inv) - rope64(x - d, pos, inv)) / 2 * w.double()).sum(-1)
        assert (grad[..., e].double() - diff).abs().max() < 1e-5


def test_rope_empty(pkg, dev):
    inv, _ = pkg.ops.rope_frequencies(64, device=dev)
    x = torch.empty((0, 4, 64), device=dev)
    assert pkg.ops.rope(x, torch.empty(0, dtype=torch.int64, device=dev), inv).shape == (0, 4, 64)


def paged(dev, dtype, kv_heads, dim, page, counts, ctx, seed, heads_first=False, slack=3):
    """Caches full of NaN, a table of pages in no order with junk behind each sequence's last page."""
    g = torch.Generator().manual_seed(seed)
    total = [n + c for n, c in zip(counts, ctx)]
    need = [-(-t // page) for t in total]
    pages = sum(need) + slack
    shape = (pages, kv_heads, page, dim) if heads_first else (pages, page, kv_heads, dim)
    kc, vc = (torch.full(shape, float("nan"), dtype=dtype, device=dev) for _ in range(2))
    if heads_first:
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    table = torch.full((len(counts), max(need + [1]) + 2), 1 << 30, dtype=torch.int32)
    order = torch.randperm(pages, generator=g).int()
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    cu = torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32)
    return kc, vc, table.to(dev), cu.to(dev), torch.tensor(total, dtype=torch.int32).to(dev)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("counts,ctx,heads,kv_heads,dim,rot,page,interleaved", [
    ([1], [0], 4, 1, 128, 128, 16, False), ([1, 1, 1], [15, 16, 17], 8, 2, 64, 64, 16, True),
    ([5, 0, 40, 1], [3, 9, 0, 70], 6, 2, 128, 64, 24, False), ([3, 2], [0, 1], 3, 3, 10, 4, 1, True),
    ([70] * 40, [0] * 40, 2, 1, 64, 0, 32, False)])
def test_kv_append(pkg, dev, dtype, heads_first, counts, ctx, heads, kv_heads, dim, rot, page, interleaved):
    kc, vc, table, cu, lengths = paged(dev, dtype, kv_heads, dim, page, counts, ctx, 3, heads_first)
    T = sum(counts) + 4  # four rows behind the last sequence
    qkv = torch.randn((T, heads + 2 * kv_heads, dim), device=dev).to(dtype)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    inv, _ = freqs(pkg, rot, dev)
    q_out = torch.full((T, heads, dim), 7.0, dtype=dtype, device=dev)
    before = kc.clone(), vc.clone()
    ret = pkg.ops.kv_append(k, v, kc, vc, table, cu, lengths, inv_freq=inv if rot else None, q=q, q_out=q_out,
                            interleaved=interleaved, mscale=1.25)
    assert ret is q_out and (q_out[sum(counts):] == 7.0).all()
    written = torch.zeros(kc.shape[:2], dtype=torch.bool, device=dev)
    at = 0
    for b, (n, c) in enumerate(zip(counts, ctx)):
        if n == 0:
            continue
        r = slice(at, at + n)
        at += n
        pos = torch.arange(c, c + n, device=dev)
        for name, got, src in (("q", q_out[r], q[r]), ("k", pages_of(kc, table, b, c + n)[c:], k[r])):
            want = rope64(src, pos, inv, interleaved, 1.25)
            check(got, want, rope_bound(src, want, inv, interleaved, 1.25), dtype)
        assert torch.equal(pages_of(vc, table, b, c + n)[c:], v[r])
        written[table[b, pos // page].long(), pos % page] = True
    for now, was in zip((kc, vc), before):
        assert torch.equal(now[~written].isnan(), was[~written].isnan())
    assert pkg._lib.device_status() == 0


def test_kv_append_own_positions_and_bad_pages(pkg, dev):
    kc, vc, table, cu, lengths = paged(dev, torch.float32, 1, 64, 8, [4, 4], [0, 6], 4)
    inv, _ = pkg.ops.rope_frequencies(64, device=dev)
    k, v = torch.randn((8, 1, 64), device=dev), torch.randn((8, 1, 64), device=dev)
    pos = torch.arange(8, device=dev) * 1000 + 5
    pkg.ops.kv_append(k, v, kc, vc, table, cu, lengths, inv_freq=inv, positions=pos)
    want = rope64(k, pos, inv)
    check(pages_of(kc, table, 0, 4), want[:4], rope_bound(k[:4], want[:4], inv), torch.float32)
    assert pkg._lib.device_status() == 0
    # pages outside the cache and positions outside the table drop their rows and say so
    for bad in (-1, kc.shape[0], 1 << 30):
        kc.fill_(9)
        t2 = table.clone()
        t2[1, 0] = bad
        pkg.ops.kv_append(k, v, kc, vc, t2, cu, lengths, inv_freq=inv)
        with pytest.raises(RuntimeError, match="page"):
            pkg._lib.check(pkg._lib.load().b2_device_status(None))
        assert int((kc != 9).any(-1).sum()) == 4 + 2  # sequence 0, and the two tokens of sequence 1 on its second page
    kc.fill_(9)
    pkg.ops.kv_append(k, v, kc, vc, table, cu, torch.tensor([2, 1 << 30], dtype=torch.int32, device=dev))
    assert pkg._lib.device_status() == pkg.ops.BAD_PAGE
    assert int((kc != 9).any(-1).sum()) == 2  # sequence 0's last two tokens
