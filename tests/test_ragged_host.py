"""The rotary, paged-cache and packed-attention wrappers without a GPU: what they refuse, the checks of the C entry
points, and the frequencies' formulas."""
import ctypes
import math

import pytest
import torch

H16 = torch.float16


@pytest.fixture
def calls(pkg, monkeypatch):
    log = []
    monkeypatch.setattr(pkg.ops, "require_cuda", lambda *tensors: None)
    monkeypatch.setattr(pkg.ops, "_launch", lambda name, device, *args: log.append((name, args + (None,))))
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: -1, raising=False)  # a CPU tensor's device index
    return log


def attn(**kw):
    a = dict(q=torch.zeros(5, 8, 64, dtype=H16), k_cache=torch.zeros(6, 16, 2, 64, dtype=H16),
             v_cache=torch.zeros(6, 16, 2, 64, dtype=H16), table=torch.zeros(2, 3, dtype=torch.int32),
             cu_q=torch.zeros(3, dtype=torch.int32), lengths=torch.zeros(2, dtype=torch.int32))
    a.update(kw)
    return a


def append(**kw):
    a = dict(k=torch.zeros(5, 2, 64, dtype=H16), v=torch.zeros(5, 2, 64, dtype=H16),
             k_cache=torch.zeros(6, 16, 2, 64, dtype=H16), v_cache=torch.zeros(6, 16, 2, 64, dtype=H16),
             table=torch.zeros(2, 3, dtype=torch.int32), cu_q=torch.zeros(3, dtype=torch.int32),
             lengths=torch.zeros(2, dtype=torch.int32))
    a.update(kw)
    return a


def test_calls_reach_the_library(pkg, calls):
    ops = pkg.ops
    assert ops.attn_paged(**attn()).shape == (5, 8, 64)
    assert ops.attn_packed(torch.zeros(5, 4, 128, dtype=H16), torch.zeros(7, 2, 128, dtype=H16),
                           torch.zeros(7, 2, 128, dtype=H16), torch.zeros(3, dtype=torch.int32),
                           torch.zeros(3, dtype=torch.int32)).shape == (5, 4, 128)
    assert ops.kv_append(**append()) is None
    assert ops.kv_append(**append(q=torch.zeros(5, 8, 64, dtype=H16))).shape == (5, 8, 64)
    assert ops.rope(torch.zeros(5, 2, 64), torch.zeros(5, dtype=torch.int64), torch.zeros(32)).shape == (5, 2, 64)
    assert [n for n, _ in calls] == ["b2_attn_ragged"] * 2 + ["b2_kv_append"] * 2 + ["b2_rope"]
    for name, args in calls[2:]:
        assert len(args) == len(pkg._lib.SIGNATURES[name][1])


BAD_ATTN = {
    "fp32 queries": dict(q=torch.zeros(5, 8, 64)), "2D queries": dict(q=torch.zeros(5, 512, dtype=H16)),
    "head dim 96": dict(q=torch.zeros(5, 8, 96, dtype=H16), k_cache=torch.zeros(6, 16, 2, 96, dtype=H16),
                        v_cache=torch.zeros(6, 16, 2, 96, dtype=H16)),
    "strided dim": dict(q=torch.zeros(5, 8, 128, dtype=H16)[..., ::2]),
    "7 heads over 2": dict(q=torch.zeros(5, 7, 64, dtype=H16)), "no heads": dict(q=torch.zeros(5, 0, 64, dtype=H16)),
    "bf16 cache": dict(k_cache=torch.zeros(6, 16, 2, 64, dtype=torch.bfloat16)),
    "unlike caches": dict(v_cache=torch.zeros(7, 16, 2, 64, dtype=H16)),
    "unlike strides": dict(v_cache=torch.zeros(6, 2, 16, 64, dtype=H16).transpose(1, 2)),
    "int64 table": dict(table=torch.zeros(2, 3, dtype=torch.int64)), "1D table": dict(table=torch.zeros(6, dtype=torch.int32)),
    "cu_q of batch": dict(cu_q=torch.zeros(2, dtype=torch.int32)), "int64 lengths": dict(lengths=torch.zeros(2, dtype=torch.int64)),
    "lengths of 3": dict(lengths=torch.zeros(3, dtype=torch.int32)), "scale 0": dict(scale=0.0),
    "negative scale": dict(scale=-1.0), "nan scale": dict(scale=math.nan), "negative cap": dict(softcap=-1.0),
    "infinite cap": dict(softcap=math.inf), "negative window": dict(window=-1), "slopes of 7": dict(slopes=torch.zeros(7)),
    "fp16 slopes": dict(slopes=torch.zeros(8, dtype=H16)), "prefix of 3": dict(prefix=torch.zeros(3, dtype=torch.int32)),
    "output shape": dict(out=torch.zeros(5, 8, 128, dtype=H16)), "output type": dict(out=torch.zeros(5, 8, 64)),
    "lse shape": dict(lse=torch.zeros(5, 2)), "small workspace": dict(workspace=torch.zeros(16, dtype=torch.uint8)),
    "pages of no rows": dict(k_cache=torch.zeros(6, 0, 2, 64, dtype=H16), v_cache=torch.zeros(6, 0, 2, 64, dtype=H16)),
}


@pytest.mark.parametrize("what", BAD_ATTN)
def test_attn_paged_refuses(pkg, calls, what):
    with pytest.raises(RuntimeError):
        pkg.ops.attn_paged(**attn(**BAD_ATTN[what]))
    assert not calls


BAD_APPEND = {
    "unlike k and v": dict(v=torch.zeros(5, 3, 64, dtype=H16)), "mixed types": dict(v=torch.zeros(5, 2, 64)),
    "fp64": dict(k=torch.zeros(5, 2, 64, dtype=torch.float64)), "cache type": dict(k_cache=torch.zeros(6, 16, 2, 64)),
    "cache heads": dict(k_cache=torch.zeros(6, 16, 3, 64, dtype=H16), v_cache=torch.zeros(6, 16, 3, 64, dtype=H16)),
    "too many pairs": dict(inv_freq=torch.zeros(33)), "fp64 inv_freq": dict(inv_freq=torch.zeros(32, dtype=torch.float64)),
    "int32 positions": dict(positions=torch.zeros(5, dtype=torch.int32)), "4 positions": dict(positions=torch.zeros(4, dtype=torch.int64)),
    "queries of 4 tokens": dict(q=torch.zeros(4, 8, 64, dtype=H16)), "q_out alone": dict(q_out=torch.zeros(5, 8, 64, dtype=H16)),
    "q_out shape": dict(q=torch.zeros(5, 8, 64, dtype=H16), q_out=torch.zeros(5, 4, 64, dtype=H16)),
    "cu_q type": dict(cu_q=torch.zeros(3, dtype=torch.int64)),
}


@pytest.mark.parametrize("what", BAD_APPEND)
def test_kv_append_refuses(pkg, calls, what):
    with pytest.raises(RuntimeError):
        pkg.ops.kv_append(**append(**BAD_APPEND[what]))
    assert not calls


def test_rope_and_packed_refuse(pkg, calls):
    ops = pkg.ops
    x, pos, inv = torch.zeros(5, 2, 64), torch.zeros(5, dtype=torch.int64), torch.zeros(32)
    for a in ((x[0], pos, inv), (x, pos[:4], inv), (x, pos.int(), inv), (x, pos, torch.zeros(33)), (x.double(), pos, inv),
              (torch.zeros(5, 2, 63), pos, inv[:8]), (torch.zeros(1, 1, 2048), pos[:1], torch.zeros(600))):
        with pytest.raises(RuntimeError):
            ops.rope(*a)
    with pytest.raises(RuntimeError, match="inv_freq"):
        ops.rope(x, pos, None)
    with pytest.raises(RuntimeError, match="output"):
        ops.rope(x, pos, inv, out=torch.zeros(5, 2, 32))
    q, k, cu = torch.zeros(5, 4, 64, dtype=H16), torch.zeros(7, 2, 64, dtype=H16), torch.zeros(3, dtype=torch.int32)
    for a in ((q, k, k[:6], cu, cu), (q, k, k, cu, cu[:2]), (q, k.float(), k.float(), cu, cu), (q, k, k, cu.long(), cu),
              (q, k[:, :0], k[:, :0], cu, cu), (q, torch.zeros(7, 2, 128, dtype=H16), torch.zeros(7, 2, 128, dtype=H16), cu, cu)):
        with pytest.raises(RuntimeError):
            ops.attn_packed(*a)
    assert not calls


def test_cpu_tensors_are_refused(pkg):
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        pkg.ops.attn_paged(**attn())
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        pkg.ops.kv_append(**append())
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        pkg.ops.rope(torch.zeros(5, 2, 64), torch.zeros(5, dtype=torch.int64), torch.zeros(32))


def test_c_entry_points_check_before_launching(pkg):
    lib, P = pkg._lib.load(), ctypes.c_void_p
    fake = P(4096)
    good = dict(q=4096, sqt=512, sqh=64, out=4096, sot=512, soh=64, lse=0, k=4096, v=4096, s_page=2048, s_row=128, s_head=64,
                table=4096, cu_q=4096, lengths=4096, prefix=0, slopes=0, workspace=4096, table_ld=3, max_pages=3, num_pages=6, page_size=16,
                batch=2, tokens=5, key_rows=6, heads=8, kv_heads=2, dim=64, dtype=0, max_q=1, causal=1, window=0, scale=0.125,
                softcap=0.0)

    def status(**kw):
        return lib.b2_attn_ragged(pkg.ops._RAGGED.pack(*{**good, **kw}.values()), P(None))

    for kw in (dict(q=0), dict(out=0), dict(k=0), dict(cu_q=0), dict(lengths=0), dict(workspace=0), dict(heads=7),
               dict(kv_heads=0), dict(batch=-1), dict(window=-1), dict(scale=0.0), dict(scale=math.nan),
               dict(softcap=-1.0), dict(page_size=0), dict(scale=math.inf)):
        assert status(**kw) == 1, kw
    for kw in (dict(dim=96), dict(dtype=2), dict(q=4098), dict(sqt=513), dict(s_row=132), dict(k=4104), dict(out=4100),
               dict(tokens=1 << 28)):
        assert status(**kw) == 2, kw
    assert status(batch=0) == 0 and status(tokens=0) == 0
    assert lib.b2_attn_ragged(None, P(None)) == 1
    assert lib.b2_attn_ragged_workspace_bytes(8, 2, 96, 1) == 0 and lib.b2_attn_ragged_workspace_bytes(8, 2, 128, 1) > 0
    turn = dict(x=4096, sxt=64, sxh=64, out=4096, sot=64, soh=64, positions=4096, inv_freq=4096, tokens=4, heads=1, dim=64,
                pairs=32, interleaved=0, dtype=0, mscale=1.0)
    rope = lambda **kw: lib.b2_rope(pkg.ops._ROPE.pack(*{**turn, **kw}.values()), P(None))
    assert [rope(x=0), rope(tokens=-1), rope(dim=63), rope(pairs=33), rope(dim=2048, pairs=1000), rope(dtype=3),
            rope(positions=0), rope(inv_freq=0), rope(tokens=0)] == [1, 1, 2, 2, 2, 2, 1, 1, 0]
    assert lib.b2_rope(None, P(None)) == 1
    block = dict(k=4096, skt=64, skh=64, v=4096, svt=64, svh=64, k_cache=4096, v_cache=4096, s_page=1024, s_row=64, s_head=64,
                 table=4096, cu_q=4096, lengths=4096, q=0, sqt=0, sqh=0, q_out=0, sot=0, soh=0, positions=0, inv_freq=4096,
                 table_ld=3, max_pages=3, num_pages=6, page_size=16, batch=2, tokens=4, heads=0, kv_heads=1, dim=64, pairs=32,
                 interleaved=0, dtype=0, mscale=1.0)
    app = lambda **kw: lib.b2_kv_append(pkg.ops._APPEND.pack(*{**block, **kw}.values()), P(None))
    assert lib.b2_kv_append(None, P(None)) == 1
    assert [app(k=0), app(page_size=0), app(heads=2), app(kv_heads=0), app(batch=0), app(tokens=0), app(dim=63), app(dtype=3),
            app(pairs=33)] == [1, 1, 1, 1, 0, 0, 2, 2, 2]


def test_rope_frequencies(pkg):
    f = pkg.ops.rope_frequencies
    d, base = 64, 10000.0
    plain = torch.tensor([base ** (-2 * i / d) for i in range(d // 2)])
    inv, ms = f(d, base)
    assert ms == 1.0 and torch.allclose(inv, plain, rtol=1e-6)
    assert torch.allclose(f(d, base, "linear", 4.0)[0], plain / 4, rtol=1e-6)
    grown, ms = f(d, base, "base", 4.0)
    assert ms == 1.0 and abs(grown[0] - 1) < 1e-6 and abs(grown[-1] / (plain[-1] / 4) - 1) < 1e-5
    ramp, ms = f(d, base, "ramp", 4.0, original_length=2048)
    assert abs(ms - (0.1 * math.log(4) + 1)) < 1e-12
    for i in range(d // 2):
        r = 2048 * base ** (-2 * i / d) / (2 * math.pi)
        keep = min(max((r - 1) / 31, 0), 1)
        assert abs(ramp[i] / (plain[i] * (keep + (1 - keep) / 4)) - 1) < 1e-5
    assert abs(ramp[0] - plain[0]) < 1e-6 and abs(ramp[-1] / plain[-1] - 0.25) < 1e-6
    for a in ((63,), (0,), (64, -1.0), (64, base, "unknown", 2.0), (64, base, None, 2.0), (64, base, "linear", 0.5),
              (64, base, "ramp", 2.0), (2, base, "base", 2.0)):
        with pytest.raises(RuntimeError):
            f(*a)
