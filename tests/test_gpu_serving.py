"""The serving operators (include/cmol_hip.h): windowed attention with sinks
for single tokens and prompts, attention behind a shared prefix, and logits for
the next token, against plain 64-bit computations.

Tolerance of an attention output: a relative error of at most e in every
softmax weight moves it by at most 2 e sum_t p_t |v_t|.  e is taken as 2^-20
(weights and queries in two halves or fp32, hardware exponential: a few 2^-23),
plus 2^-20 of the row's largest sum_d |q_d k_d| / sqrt(d_head) (a score is an
fp32 sum of up to 256 products: sqrt(256) 2^-24), plus sqrt(T) 2^-24 for the
sums over T positions."""
import ctypes as C
import threading

import numpy as np
import pytest

from libcmol_amd import hiprt, native

pytestmark = pytest.mark.gpu
F32, F16 = 0, 1


@pytest.fixture(scope="module")
def ctx(gpu):
    c = gpu.Ctx(1 << 30)
    yield c
    c.close()


def reference(q, k, v, seen):
    """q [h][d]; k, v [kv][T][d] 64-bit; seen [T]: outputs [h][d] and their tolerance."""
    h, d = q.shape
    kv = k.shape[0]
    out, tol = np.zeros((h, d)), np.zeros((h, d))
    t = np.flatnonzero(seen)
    if len(t) == 0:
        return out, tol
    for i in range(h):
        kk, vv = k[i * kv // h][t], v[i * kv // h][t]
        s = kk @ q[i] / np.sqrt(d)
        p = np.exp(s - s.max())
        p /= p.sum()
        out[i] = p @ vv
        a = (np.abs(kk) @ np.abs(q[i])).max() / np.sqrt(d)
        e = 2.0**-20 + a * 2.0**-20 + np.sqrt(len(t)) * 2.0**-24
        tol[i] = 2 * e * (p @ np.abs(vv)) + 1e-30
    return out, tol


def rand_cache(rng, shape, f16):
    x = rng.standard_normal(shape).astype(np.float32)
    return x.astype(np.float16) if f16 else x


def guarded(ctx, nbytes):
    """A device buffer of nbytes with a canary behind it."""
    d = ctx.alloc(nbytes + 256)
    ctx.h2d(d + nbytes, np.full(256, 0xA5, np.uint8))
    return d


def canary(ctx, d, nbytes):
    return np.all(ctx.d2h(d + nbytes, 256, np.uint8) == 0xA5)


def room(ctx, need):
    """A workspace of exactly `need` bytes, full of NaN, with a canary."""
    assert need > 0
    ws = guarded(ctx, need)
    ctx.h2d(ws, np.full(need, 0xFF, np.uint8))
    return ws


def p(x):
    return C.c_void_p(x)


def close(got, want, tol, what):
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(got - want) / (tol + 1e-30)):.3g} x tol"


def window_call(ctx, q, dk, dv, slots, stride, lens, heads, kv, dh, max_ctx, f16, window, sinks, n=None):
    L = native.lib()
    n = n or len(lens)
    need = L.cmolhip_attn_window_bytes(n, heads, kv, dh, max_ctx, window, sinks)
    ws, out = room(ctx, need), guarded(ctx, n * heads * dh * 4)
    ctx.h2d(out, np.full(n * heads * dh, 777.0, np.float32))
    dq, dl = ctx.upload(q), ctx.upload(np.array(lens, np.int32))
    ds = ctx.upload(np.array(slots, np.int32)) if slots is not None else None
    native.check(L.cmolhip_attn_window(ctx.h, n, p(dq), p(dk), p(dv), p(ds), stride, p(dl), heads, kv, dh, max_ctx, f16,
                                       window, sinks, p(ws), need, p(out)), "window")
    native.check(L.cmolhip_synchronize(ctx.h), "sync")
    assert canary(ctx, ws, need) and canary(ctx, out, n * heads * dh * 4)
    return ctx.d2h(out, (n, heads, dh), np.float32)


def window_seen(L, max_ctx, window, sinks):
    L = max(0, min(L, max_ctx))
    t = np.arange(max_ctx)
    return (t < L) & ((t < sinks) | (t >= L - window))


WINDOW_CASES = [
    # heads, kv, d_head, max_ctx, lengths (0 and below: nothing; past max_ctx: max_ctx), window, sinks
    (9, 3, 64, 700, [1, 2, 3, 5, 131, 132, 133, 700], 128, 4),
    (16, 4, 128, 1100, [1100, 64, 33, 0, 17, 1099, 5000, -3], 300, 1),
    (16, 4, 128, 400, [400, 1, 40], 1, 0), (16, 4, 128, 400, [400, 1, 40, 0], 1, 1),
    (4, 4, 16, 300, [300, 7, 100], 33, 5), (8, 1, 32, 513, [513, 512, 31], 100, 33),
    (8, 2, 256, 260, [260, 77, 1], 64, 2), (6, 6, 256, 200, [200, 3], 1 << 30, 0),
    (32, 1, 64, 333, [333, 12, 0], 90, 4), (20, 2, 128, 270, [270, 269], 50, 64), (34, 2, 32, 90, [90, 5], 30, 3),
    (8, 2, 64, 500, [500, 20, 499], 2**31 - 1, 0), (8, 2, 64, 500, [500, 20, 499], 7, 2**31 - 1),
    (8, 2, 64, 500, [500, 20, 499], 2**31 - 1, 2**31 - 1), (15, 5, 64, 2000, [2000, 64, 1000, 601, 602, 603], 601, 1),
    (2, 1, 128, 5000, [5000, 4999], 4000, 64), (1, 1, 64, 37, [37], 5, 0),
    (3, 3, 128, 64, [int(x) for x in np.random.default_rng(3).integers(0, 65, 70)], 20, 3),
    # long contexts in balanced ranges: one item, more items than a wave has lanes, items of nothing among them
    (2, 1, 64, 3000, [2999], 2500, 40), (4, 1, 64, 1500, [int(x) for x in np.random.default_rng(4).integers(-5, 1501, 100)], 1200, 4),
    (6, 3, 128, 2100, [2100, 0, 1500, 3, 2099, 0], 1700, 100), (2, 2, 256, 1400, [1400, 700], 1300, 0),
    (16, 2, 16, 1300, [1300, 1299, 64], 1100, 9), (8, 1, 32, 1300, [1300, 31], 1290, 5),
]


def session_form(monkeypatch, form):
    """Sessions in pieces ("0"), whole ("1"), or (None) as estimated."""
    if form is None:
        monkeypatch.delenv("CMOL_SESSION_WHOLE", raising=False)
    else:
        monkeypatch.setenv("CMOL_SESSION_WHOLE", form)


@pytest.mark.parametrize("form", [None, "0", "1"])
@pytest.mark.parametrize("f16", [F32, F16])
@pytest.mark.parametrize("heads,kv,dh,max_ctx,lens,window,sinks", WINDOW_CASES, ids=str)
def test_window_against_64_bits(ctx, monkeypatch, heads, kv, dh, max_ctx, lens, window, sinks, f16, form):
    """Every position that no row sees holds NaN or an infinity; queries of
    half of the rows are large, so their softmaxes are peaked."""
    session_form(monkeypatch, form)
    c = native.Ctx(256 << 20)
    rng = np.random.default_rng(heads * dh + len(lens))
    n = len(lens)
    q = rng.standard_normal((n, heads, dh)).astype(np.float32)
    q[::2] *= 6
    k, v = (rand_cache(rng, (n, kv, max_ctx, dh), f16) for _ in range(2))
    seen = [window_seen(x, max_ctx, window, sinks) for x in lens]
    junk = [np.nan, np.inf, -np.inf]
    for i in range(n):
        k[i][:, ~seen[i]] = junk[i % 3]
        v[i][:, ~seen[i]] = junk[(i + 1) % 3]
    got = window_call(c, q, c.upload(k), c.upload(v), None, 0, lens, heads, kv, dh, max_ctx, f16, window, sinks)
    for i in range(n):
        want, tol = reference(q[i].astype(np.float64), k[i].astype(np.float64), v[i].astype(np.float64), seen[i])
        close(got[i], want, tol, f"session {i}, length {lens[i]}")
    c.close()


@pytest.mark.parametrize("form", [None, "0", "1"])
@pytest.mark.parametrize("f16", [F32, F16])
@pytest.mark.parametrize("heads,kv,dh", [(16, 4, 128), (9, 3, 64), (16, 1, 64), (16, 2, 128), (8, 2, 256)])
def test_window_of_many_long_sessions(ctx, monkeypatch, heads, kv, dh, f16, form):
    """More than 110 MB that a call may read (sessions share three caches, which
    read as many bytes)."""
    session_form(monkeypatch, form)
    c = native.Ctx(256 << 20)
    n, max_ctx, window, sinks = 100, 6000, 5000, 4
    rng = np.random.default_rng(heads + dh)
    slots = rng.integers(0, 3, n).astype(np.int32)
    lens = rng.integers(0, 400, n).astype(np.int32)
    lens[:4], slots[5] = [6000, 5003, 1, 2000], -1
    assert 2 * n * (window + sinks) * kv * dh * (2 if f16 else 4) > 110e6
    q = rng.standard_normal((n, heads, dh)).astype(np.float32)
    k, v = (rand_cache(rng, (3, kv, max_ctx, dh), f16) for _ in range(2))
    got = window_call(c, q, c.upload(k), c.upload(v), slots, 0, lens, heads, kv, dh, max_ctx, f16, window, sinks)
    for i in range(n):
        seen = window_seen(lens[i] if slots[i] >= 0 else 0, max_ctx, window, sinks)
        want, tol = reference(q[i].astype(np.float64), k[slots[i]].astype(np.float64), v[slots[i]].astype(np.float64), seen)
        close(got[i], want, tol, f"session {i}")
    c.close()


@pytest.mark.parametrize("f16", [F32, F16])
def test_window_over_slots_of_a_pool(ctx, f16):
    """Sessions in any slot, one of them twice, padding (slot -1), caches
    further apart than they are long (the other layers' positions between)."""
    heads, kv, dh, max_ctx, window, sinks = 8, 2, 64, 300, 90, 3
    stride = 3 * kv * max_ctx * dh
    rng = np.random.default_rng(8)
    pool_k, pool_v = (rand_cache(rng, (4, 3, kv, max_ctx, dh), f16) for _ in range(2))
    for x in (pool_k, pool_v):
        x[:, 0], x[:, 2] = np.nan, np.nan
    slots, lens = [3, -1, 0, 1, 1], [300, 200, 5, 91, 93]
    q = rng.standard_normal((5, heads, dh)).astype(np.float32)
    size = kv * max_ctx * dh * (2 if f16 else 4)   # the middle layer
    got = window_call(ctx, q, ctx.upload(pool_k) + size, ctx.upload(pool_v) + size, slots, stride, lens, heads, kv, dh,
                      max_ctx, f16, window, sinks)
    for i, s in enumerate(slots):
        if s < 0:
            assert np.all(got[i] == 0)
            continue
        want, tol = reference(q[i].astype(np.float64), pool_k[s, 1].astype(np.float64), pool_v[s, 1].astype(np.float64),
                              window_seen(lens[i], max_ctx, window, sinks))
        close(got[i], want, tol, f"session {i}")


def prompt_call(ctx, q, dk, dv, pos0, heads, kv, dh, max_ctx, f16, window, sinks):
    L = native.lib()
    n = len(q)
    need = L.cmolhip_attn_window_prompt_bytes(n, heads, kv, dh, max_ctx, window, sinks)
    ws, out = room(ctx, need), guarded(ctx, n * heads * dh * 4)
    ctx.h2d(out, np.full(n * heads * dh, 777.0, np.float32))
    dq = ctx.upload(q)
    native.check(L.cmolhip_attn_window_prompt(ctx.h, n, pos0, p(dq), p(dk), p(dv), heads, kv, dh, max_ctx, f16, window,
                                              sinks, p(ws), need, p(out)), "prompt")
    native.check(L.cmolhip_synchronize(ctx.h), "sync")
    assert canary(ctx, ws, need) and canary(ctx, out, n * heads * dh * 4)
    return ctx.d2h(out, (n, heads, dh), np.float32)


PROMPT_CASES = [
    # heads, kv, d_head, n, pos0, max_ctx, window, sinks
    (9, 3, 64, 1, 0, 10, 4, 0), (9, 3, 64, 45, 333, 400, 256, 4), (16, 4, 128, 130, 0, 130, 64, 4),
    (16, 4, 128, 33, 700, 1000, 1, 0), (16, 4, 128, 65, 31, 100, 1, 1), (4, 4, 16, 77, 5, 100, 20, 7),
    (8, 1, 32, 100, 60, 160, 33, 50), (8, 2, 256, 40, 30, 90, 25, 2), (32, 1, 64, 19, 100, 200, 64, 3),
    (20, 2, 128, 23, 9, 40, 2**31 - 1, 0), (6, 2, 64, 50, 10, 70, 8, 2**31 - 1), (15, 5, 64, 300, 250, 600, 120, 64),
    (3, 3, 128, 200, 0, 256, 100, 0), (5, 1, 64, 64, 64, 128, 32, 0),
    # sinks of more than a tile, apart from the window, met by it and reaching into it; a window of everything
    (16, 4, 128, 150, 900, 1100, 500, 70), (16, 4, 128, 260, 0, 300, 100, 70), (15, 5, 64, 333, 100, 500, 64, 300),
    (16, 4, 128, 140, 150, 300, 100, 200), (8, 2, 64, 700, 0, 700, 5000, 0), (4, 1, 128, 129, 63, 256, 65, 64),
    (2, 1, 64, 32, 0, 32, 1, 0), (2, 1, 128, 33, 31, 64, 33, 31),
]


def prompt_form(monkeypatch, form):
    """The prompt's form: None the estimated one, "0" 16-row work-groups, "1"
    128-row ones that share the positions through LDS."""
    if form is None:
        monkeypatch.delenv("CMOL_WINDOW_PROMPT", raising=False)
    else:
        monkeypatch.setenv("CMOL_WINDOW_PROMPT", form)


@pytest.mark.parametrize("form", [None, "0", "1"])
@pytest.mark.parametrize("f16", [F32, F16])
@pytest.mark.parametrize("heads,kv,dh,n,pos0,max_ctx,window,sinks", PROMPT_CASES, ids=str)
def test_prompt_against_64_bits(ctx, monkeypatch, heads, kv, dh, n, pos0, max_ctx, window, sinks, f16, form):
    prompt_form(monkeypatch, form)
    c = native.Ctx(256 << 20)
    rng = np.random.default_rng(heads * dh + n)
    q = rng.standard_normal((n, heads, dh)).astype(np.float32)
    q[::2] *= 6
    k, v = (rand_cache(rng, (kv, max_ctx, dh), f16) for _ in range(2))
    seen = [window_seen(pos0 + i + 1, max_ctx, window, sinks) for i in range(n)]
    unseen = ~np.any(seen, axis=0)
    k[:, unseen], v[:, unseen] = np.nan, np.inf
    got = prompt_call(c, q, c.upload(k), c.upload(v), pos0, heads, kv, dh, max_ctx, f16, window, sinks)
    for i in range(n):
        want, tol = reference(q[i].astype(np.float64), k.astype(np.float64), v.astype(np.float64), seen[i])
        close(got[i], want, tol, f"token {i}")
    c.close()


@pytest.mark.parametrize("form", ["0", "1"])
@pytest.mark.parametrize("f16", [F32, F16])
@pytest.mark.parametrize("heads,kv,dh", [(16, 4, 128), (9, 3, 64), (4, 4, 32)])
def test_prompt_positions_that_are_not_finite(ctx, monkeypatch, heads, kv, dh, f16, form):
    """NaN and infinities in positions that some tokens see and others mask:
    the tokens that do not see one come out as without it."""
    prompt_form(monkeypatch, form)
    n, pos0, max_ctx, window, sinks = 90, 40, 160, 30, 2
    rng = np.random.default_rng(2)
    q = rng.standard_normal((n, heads, dh)).astype(np.float32)
    k, v = (rand_cache(rng, (kv, max_ctx, dh), f16) for _ in range(2))
    bad = [50, 77, 78, 100, 128]
    v[:, 50], v[0, 77], k[:, 78], v[:, 100, 3], k[0, 128, 0] = np.inf, np.nan, np.nan, -np.inf, np.inf
    got = prompt_call(ctx, q, ctx.upload(k), ctx.upload(v), pos0, heads, kv, dh, max_ctx, f16, window, sinks)
    for i in range(n):
        seen = window_seen(pos0 + i + 1, max_ctx, window, sinks)
        if seen[bad].any():
            assert not np.all(np.isfinite(got[i])), f"token {i} sees a value that is not finite"
            continue
        want, tol = reference(q[i].astype(np.float64), k.astype(np.float64), v.astype(np.float64), seen)
        close(got[i], want, tol, f"token {i}")


@pytest.mark.parametrize("form", ["0", "1"])
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("k_scale,v_scale", [(1e-6, 1e-6), (1e-3, 1e9), (1e-30, 1e-30), (1e3, 1.0), (1.0, 1e30)])
def test_prompt_over_caches_of_any_range(ctx, monkeypatch, dh, k_scale, v_scale, form):
    """fp32 caches far from 1, each position's row times another power of ten
    up to 10^4; the queries make up for K, so the scores are ordinary.  The
    absolute term: a value of a tile of 32 positions is held to 2^-33 of the
    tile's largest."""
    prompt_form(monkeypatch, form)
    heads, kv, n, pos0, max_ctx, window, sinks = 8, 2, 70, 100, 200, 90, 5
    rng = np.random.default_rng(int(dh + np.log10(v_scale)))
    q = (rng.standard_normal((n, heads, dh)) / k_scale / 1e3).astype(np.float32)
    k = (rng.standard_normal((kv, max_ctx, dh)) * k_scale * 10 ** rng.uniform(0, 4, (kv, max_ctx, 1))).astype(np.float32)
    v = (rng.standard_normal((kv, max_ctx, dh)) * v_scale * 10 ** rng.uniform(0, 4, (kv, max_ctx, 1))).astype(np.float32)
    got = prompt_call(ctx, q, ctx.upload(k), ctx.upload(v), pos0, heads, kv, dh, max_ctx, 0, window, sinks)
    for i in range(n):
        seen = window_seen(pos0 + i + 1, max_ctx, window, sinks)
        want, tol = reference(q[i].astype(np.float64), k.astype(np.float64), v.astype(np.float64), seen)
        close(got[i] / v_scale, want / v_scale, tol / v_scale + 2.0**-33 * np.abs(v / v_scale).max(), f"token {i}")


@pytest.mark.parametrize("form", ["0", "1"])
@pytest.mark.parametrize("f16", [F32, F16])
@pytest.mark.parametrize("heads,kv,dh", [(16, 4, 128), (9, 3, 64), (4, 4, 32)])
@pytest.mark.parametrize("big,small", [(1e18, 1e-9), (1e30, 1e-30), (6e4, 1e-3), (3e3, 1.0)])
def test_prompt_large_values_elsewhere(ctx, monkeypatch, heads, kv, dh, f16, form, big, small):
    """Finite but large K and V rows, next to ordinary ones and next to rows
    of small values: tokens that do not see them, or give them no weight, come
    out as without them.  Every query has 3 in its first dimension, so `low`
    scores -3 big / sqrt(d_head), a weight of exp(-500) and less, 0.  Absolute
    term: a V row is held to 2^-33 of its largest."""
    prompt_form(monkeypatch, form)
    n, pos0, max_ctx, window, sinks = 90, 40, 160, 30, 2
    rng = np.random.default_rng(11)
    q = rng.standard_normal((n, heads, dh)).astype(np.float32)
    q[..., 0] = 3
    k, v = (rand_cache(rng, (kv, max_ctx, dh), f16) for _ in range(2))
    if f16:
        big, small = min(big, 6e4), max(small, 1e-3)
    low, seen_big = [45, 88, 110], [0, 60, 99, 129]
    v[:, 20:28] *= v.dtype.type(small)
    v[:, 70:75] *= v.dtype.type(small)
    k[:, 84:86] *= k.dtype.type(small)
    k[:, 112], v[:, 114] = 0, 0
    k[:, low] = 0
    k[:, low, 0] = -big
    v[:, low] = np.sign(v[:, low]) * v.dtype.type(big)
    v[:, seen_big[1:]] = np.sign(v[:, seen_big[1:]]) * v.dtype.type(big)
    got = prompt_call(ctx, q, ctx.upload(k), ctx.upload(v), pos0, heads, kv, dh, max_ctx, f16, window, sinks)
    k64, v64 = k.astype(np.float64), v.astype(np.float64)
    for i in range(n):
        seen = window_seen(pos0 + i + 1, max_ctx, window, sinks)
        seen[low] = False
        want, tol = reference(q[i].astype(np.float64), k64, v64, seen)
        tops = np.repeat(np.abs(v64).max(2, keepdims=True), dh, 2)
        for h in range(heads):
            s = k64[h * kv // heads][seen] @ q[i, h].astype(np.float64) / np.sqrt(dh)
            w = np.exp(s - s.max())
            tol[h] += 2.0**-33 * (w / w.sum()) @ tops[h * kv // heads][seen]
        close(got[i], want, tol, f"token {i}")


def test_prompt_tokens_equal_single_tokens(ctx):
    """A prompt's rows and the same tokens decoded one by one, as sessions
    over one cache."""
    heads, kv, dh, n, pos0, max_ctx, window, sinks = 16, 4, 128, 21, 200, 300, 100, 4
    rng = np.random.default_rng(4)
    q = rng.standard_normal((n, heads, dh)).astype(np.float32)
    k, v = (rand_cache(rng, (kv, max_ctx, dh), 1) for _ in range(2))
    dk, dv = ctx.upload(k), ctx.upload(v)
    a = prompt_call(ctx, q, dk, dv, pos0, heads, kv, dh, max_ctx, 1, window, sinks)
    b = window_call(ctx, q, dk, dv, [0] * n, 0, list(range(pos0 + 1, pos0 + n + 1)), heads, kv, dh, max_ctx, 1, window, sinks)
    assert np.max(np.abs(a - b)) < 1e-5


def shared_call(ctx, q, dpk, dpv, prefix, prefix_ctx, dk, dv, slots, stride, lens, heads, kv, dh, max_ctx, f16):
    L = native.lib()
    n = len(lens)
    need = L.cmolhip_attn_shared_bytes(n, heads, kv, dh, prefix, max_ctx)
    ws, out = room(ctx, need), guarded(ctx, n * heads * dh * 4)
    ctx.h2d(out, np.full(n * heads * dh, 777.0, np.float32))
    dq, dl = ctx.upload(q), ctx.upload(np.array(lens, np.int32))
    ds = ctx.upload(np.array(slots, np.int32)) if slots is not None else None
    native.check(L.cmolhip_attn_shared(ctx.h, n, p(dq), p(dpk), p(dpv), prefix, prefix_ctx, p(dk), p(dv), p(ds), stride,
                                       p(dl), heads, kv, dh, max_ctx, f16, p(ws), need, p(out)), "shared")
    native.check(L.cmolhip_synchronize(ctx.h), "sync")
    assert canary(ctx, ws, need) and canary(ctx, out, n * heads * dh * 4)
    return ctx.d2h(out, (n, heads, dh), np.float32)


SHARED_CASES = [
    # heads, kv, d_head, prefix, room for it, lengths, max_ctx
    (9, 3, 64, 777, 777, [8, 250, 33, 0, 1], 256), (16, 4, 128, 1, 64, [1, 0], 32), (16, 4, 128, 0, 16, [5, 0, 300], 300),
    (16, 4, 128, 2000, 2048, [16, 500, 64, 65, 63, 128, 1, 2, 3], 500), (16, 4, 128, 300, 300, [40], 64),
    (4, 4, 16, 100, 120, [9, 30], 30), (8, 1, 32, 257, 300, [100, 31, 0, -4], 100), (8, 2, 256, 130, 130, [70, 1, 20], 70),
    (32, 1, 64, 95, 96, [33, 2, 64], 64), (20, 2, 128, 64, 64, [5000, 12], 31), (34, 2, 32, 31, 40, [5, 6], 8),
    (15, 5, 64, 513, 600, [int(x) for x in np.random.default_rng(5).integers(0, 90, 70)], 90),
    (2, 1, 64, 5000, 5000, [1, 700], 700), (1, 1, 128, 33, 33, [0], 4), (8, 8, 64, 200, 256, [10, 20, 30], 40),
    # own contexts in balanced ranges, more sessions than a wave has lanes
    (4, 2, 64, 300, 300, [int(x) for x in np.random.default_rng(6).integers(-5, 400, 100)], 400),
    (16, 4, 128, 100, 128, [900, 0, 31, 899], 900), (4, 2, 256, 70, 70, [600, 3, 0], 600),
    # a long prefix before a few rows: many parts
    (4, 1, 64, 9000, 9000, [3, 0], 16), (2, 1, 16, 20000, 20000, [40], 64),
    # two row tiles a work-group at the smallest d_head
    (16, 2, 16, 200, 200, [30, 5, 0, 64], 64),
]


@pytest.mark.parametrize("form", [None, "0", "1"])
@pytest.mark.parametrize("f16", [F32, F16])
@pytest.mark.parametrize("heads,kv,dh,prefix,prefix_ctx,lens,max_ctx", SHARED_CASES, ids=str)
def test_shared_against_64_bits(ctx, monkeypatch, heads, kv, dh, prefix, prefix_ctx, lens, max_ctx, f16, form):
    """By the estimated form, the prefix read once for all ("0"), and every session
    by itself ("1")."""
    session_form(monkeypatch, form)
    c = native.Ctx(256 << 20)
    rng = np.random.default_rng(heads * dh + prefix)
    n = len(lens)
    q = rng.standard_normal((n, heads, dh)).astype(np.float32)
    q[::2] *= 6
    pk, pv = (rand_cache(rng, (kv, prefix_ctx, dh), f16) for _ in range(2))
    k, v = (rand_cache(rng, (n, kv, max_ctx, dh), f16) for _ in range(2))
    pk[:, prefix:], pv[:, prefix:] = np.nan, np.inf
    own = [max(0, min(x, max_ctx)) for x in lens]
    for i in range(n):
        k[i][:, own[i]:], v[i][:, own[i]:] = np.inf, np.nan
    got = shared_call(c, q, c.upload(pk), c.upload(pv), prefix, prefix_ctx, c.upload(k), c.upload(v), None, 0, lens, heads,
                      kv, dh, max_ctx, f16)
    for i in range(n):
        kk = np.concatenate([pk[:, :prefix], k[i][:, :own[i]]], 1).astype(np.float64)
        vv = np.concatenate([pv[:, :prefix], v[i][:, :own[i]]], 1).astype(np.float64)
        want, tol = reference(q[i].astype(np.float64), kk, vv, np.ones(kk.shape[1], bool))
        close(got[i], want, tol, f"session {i}, length {lens[i]}")
    c.close()


@pytest.mark.parametrize("f16", [F32, F16])
def test_shared_prefix_in_a_slot_of_the_pool(ctx, f16):
    """The prefix is the start of one session's own cache, that session goes
    on behind it elsewhere; padding sees the prefix alone; a session twice."""
    heads, kv, dh, max_ctx, prefix = 8, 2, 64, 200, 70
    rng = np.random.default_rng(9)
    pk, pv = (rand_cache(rng, (5, kv, max_ctx, dh), f16) for _ in range(2))
    slots, lens = [4, 1, -1, 2, 1], [3, 150, 10, 0, 149]
    q = rng.standard_normal((5, heads, dh)).astype(np.float32)
    dk, dv = ctx.upload(pk), ctx.upload(pv)
    got = shared_call(ctx, q, dk, dv, prefix, max_ctx, dk, dv, slots, 0, lens, heads, kv, dh, max_ctx, f16)
    for i, s in enumerate(slots):
        m = lens[i] if s >= 0 else 0
        kk = np.concatenate([pk[0][:, :prefix], pk[s][:, :m]], 1).astype(np.float64)
        vv = np.concatenate([pv[0][:, :prefix], pv[s][:, :m]], 1).astype(np.float64)
        want, tol = reference(q[i].astype(np.float64), kk, vv, np.ones(prefix + m, bool))
        close(got[i], want, tol, f"session {i}")


# ---- logits -------------------------------------------------------------------------------

def logits_reference(x, hist, rep, frq, prs, bias, allowed):
    """Row by row in fp32 with the host sampler's penalty; the choice."""
    x = x.copy()
    V = len(x)
    ids = np.array([t for t in hist if 0 <= t < V], np.int32)
    if rep is not None and len(ids):
        native.lib().cmol_apply_repeat_penalty(native.ptr(x), V, native.ptr(ids), len(ids), C.c_float(rep))
    for t, c in zip(*np.unique(ids, return_counts=True)):
        x[t] = x[t] - (np.float32(frq) * np.float32(c) + np.float32(prs))
    for t, b in dict(bias).items():
        if 0 <= t < V:
            x[t] += np.float32(b)
    if allowed is not None:
        x[~allowed] = -np.inf
    ok = x > -np.inf
    return x, int(np.argmax(np.where(ok, x, -np.inf))) if ok.any() else -1


def words_of(allowed):
    m, V = allowed.shape
    pad = np.zeros((m, (V + 31) // 32 * 32), np.uint8)
    pad[:, :V] = allowed
    pad[:, V:] = 1   # bits past the vocabulary say nothing
    return np.packbits(pad, axis=1, bitorder="little").view(np.uint32)


def logits_call(ctx, x, hist=None, rep=None, frq=None, prs=None, bias=None, allowed=None, mask_row=None, stride=None,
                inplace=False, want_out=True, want_next=True):
    L = native.lib()
    n, V = x.shape
    stride = stride or V
    rows = np.full((n, stride), 123.0, np.float32)
    rows[:, :V] = x
    d = native.Logits()
    d.n, d.vocab, d.stride = n, V, stride
    d.logits = ctx.upload(rows)
    out = d.logits if inplace else ctx.upload(np.full((n, stride), 55.0, np.float32))
    d.out = out if want_out else None
    nxt = guarded(ctx, n * 4)
    d.next = nxt if want_next else None
    if hist is not None:
        cap = max(len(h) for h in hist)
        d.history = ctx.upload(np.array([list(h) + [0] * (cap - len(h)) for h in hist], np.int32).reshape(n, cap))
        d.history_len, d.history_cap = ctx.upload(np.array([len(h) for h in hist], np.int32)), cap
    if bias is not None:
        cap = max(len(b) for b in bias)
        d.bias_ids = ctx.upload(np.array([[t for t, _ in b] + [0] * (cap - len(b)) for b in bias], np.int32).reshape(n, cap))
        d.bias = ctx.upload(np.array([[v for _, v in b] + [9.0] * (cap - len(b)) for b in bias], np.float32).reshape(n, cap))
        d.bias_len, d.bias_cap = ctx.upload(np.array([len(b) for b in bias], np.int32)), cap
    for f, a in (("repeat", rep), ("frequency", frq), ("presence", prs)):
        if a is not None:
            setattr(d, f, ctx.upload(np.array(a, np.float32)))
    if allowed is not None:
        d.mask, d.mask_rows = ctx.upload(words_of(allowed)), len(allowed)
        if mask_row is not None:
            d.mask_row = ctx.upload(np.array(mask_row, np.int32))
    need = L.cmolhip_logits_bytes(n, V)
    ws = room(ctx, need)
    native.check(L.cmolhip_logits(ctx.h, C.byref(d), p(ws), need), "logits")
    native.check(L.cmolhip_synchronize(ctx.h), "sync")
    assert canary(ctx, ws, need) and canary(ctx, nxt, n * 4)
    got = ctx.d2h(out, (n, stride), np.float32)
    assert np.all(got[:, V:] == (123.0 if inplace else 55.0))
    return got[:, :V], ctx.d2h(nxt, n, np.int32)


@pytest.mark.parametrize("n,V", [(1, 1), (1, 31), (3, 33), (2, 2047), (5, 2048), (2, 2049), (4, 5001), (1, 49152), (7, 20000)])
@pytest.mark.parametrize("inplace", [False, True])
def test_logits_against_the_host(ctx, n, V, inplace):
    """All parts at once, bit for bit (every step is one fp32 operation)."""
    rng = np.random.default_rng(n * V)
    x = (3 * rng.standard_normal((n, V))).astype(np.float32)
    hist = [list(rng.integers(-2, V + 3, m)) + [int(V // 2)] * 5 for m in rng.integers(0, 300, n)]
    rep, frq, prs = rng.uniform(0.9, 1.5, n), rng.uniform(0, 0.3, n), rng.uniform(-0.2, 0.5, n)
    rep, frq, prs = (a.astype(np.float32) for a in (rep, frq, prs))
    bias = [[(int(t), float(np.float32(b))) for t, b in zip(rng.integers(-1, V + 2, m), 4 * rng.standard_normal(m))]
            for m in rng.integers(0, 40, n)]
    allowed = rng.random((3, V)) < np.array([[0.02], [0.5], [0.9]])
    mask_row = [int(t) for t in rng.integers(-2, 4, n)]
    got, nxt = logits_call(ctx, x, hist, rep, frq, prs, bias, allowed, mask_row, stride=V + 5, inplace=inplace)
    for i in range(n):
        ok = allowed[mask_row[i]] if 0 <= mask_row[i] < 3 else None
        want, best = logits_reference(x[i], hist[i], rep[i], frq[i], prs[i], bias[i], ok)
        assert np.array_equal(got[i].view(np.uint32), want.view(np.uint32)), f"row {i}"
        assert nxt[i] == best, f"row {i}"


@pytest.mark.parametrize("n", [2, 17])
def test_logits_of_words_repeated_often(ctx, n):
    """1 to 500 occurrences of a word, penalties from 1 + 2^-23 to 1e9: bit for
    bit the host's, one division or product after the other; few and many rows
    (small and large slabs)."""
    V = 140000
    rng = np.random.default_rng(n)
    x = (10.0 ** rng.uniform(-40, 30, (n, V)) * rng.choice([-1, 1], (n, V))).astype(np.float32)
    x[:, :2000] = (5 * rng.standard_normal((n, 2000))).astype(np.float32)
    ids = rng.permutation(2000)[:40].tolist() + rng.integers(0, V, 20).tolist()
    counts = rng.integers(1, 500, 60)
    hist = [rng.permutation(np.repeat(ids, counts)).tolist() for _ in range(n)]
    rep = [[1.1, 1.0 + 2.0**-23, 1.5, 2.0, 16.0, 1e9, 1.0001, np.float32(2) - np.float32(2.0**-23)][i % 8] for i in range(n)]
    got, nxt = logits_call(ctx, x, hist=hist, rep=rep)
    for i in range(n):
        want, best = logits_reference(x[i], hist[i], rep[i], 0, 0, [], None)
        assert np.array_equal(got[i].view(np.uint32), want.view(np.uint32)), f"row {i}"
        assert nxt[i] == best, f"row {i}"


def test_logits_edges(ctx):
    """A row without an allowed token, ties, infinities and NaN, a token
    repeated past every range, an id listed twice, empty lists."""
    V = 4100
    x = np.zeros((8, V), np.float32)
    x[0] = 1.0                                   # nothing allowed
    x[1, [5, 2050, 4099]] = 7.0                  # a tie
    x[2] = np.nan                                # only NaN
    x[3, 10], x[3, 20], x[3, 3000] = np.nan, 2.0, np.inf
    x[4] = -np.inf                               # nothing above -inf
    x[5, 0] = -0.0                               # equal to the zeros behind it
    x[6, 3] = 3e38                               # repeated until it underflows, and past -inf below
    x[6, 4] = -3e38
    x[7] = -5.0
    hist = [[], [5], [1], [20], [], [], [3] * 3000 + [4] * 3000, []]
    rep = [1.1, 1.5, 1.2, 1.1, 1.1, 1.1, 1.3, 1.0]
    allowed = np.ones((8, V), bool)
    allowed[0] = False
    bias = [[], [], [], [], [], [], [], [(7, 100.0), (9, 2.0), (7, -1.0)]]
    got, nxt = logits_call(ctx, x, hist=hist, rep=rep, bias=bias, allowed=allowed)
    assert nxt.tolist() == [-1, 2050, -1, 3000, -1, 0, 3, 9]
    assert np.all(got[0] == -np.inf) and np.all(np.isnan(got[2])) and got[1, 5] == np.float32(7.0) / np.float32(1.5)
    # (fp32 division stops at two steps above 0: 2 / 1.3 = 1.54 rounds to 2)
    assert got[6, 3] == np.float32(2 * 2.0**-149) and got[6, 4] == -np.inf and got[7, 7] == -6.0 and got[7, 9] == -3.0


def test_logits_parts_left_out(ctx):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((3, 3000)).astype(np.float32)
    got, nxt = logits_call(ctx, x)
    assert np.array_equal(got, x) and np.array_equal(nxt, x.argmax(1))
    got, nxt = logits_call(ctx, x, want_out=False)
    assert np.all(got == 55.0) and np.array_equal(nxt, x.argmax(1))
    got, _ = logits_call(ctx, x, hist=[[1, 1], [], [2]], frq=[0.5, 0.5, 0.5], want_next=False)
    assert got[0, 1] == x[0, 1] - np.float32(1.0) and got[2, 2] == x[2, 2] - np.float32(0.5)


# ---- all of them --------------------------------------------------------------------------

def test_refusals(ctx):
    """A refused call launches nothing: its output stays as it was."""
    L = native.lib()
    d = ctx.alloc(1 << 20)
    out = ctx.upload(np.full(1024, 5.0, np.float32))
    A = native.CMOL_ERR_ARGS
    ws = 1 << 19

    def win(c=ctx.h, n=1, q=d, k=d, v=d, slots=None, stride=0, lens=d, heads=4, kv=2, dh=64, ctx_=8, win_=4, sinks=1, ws_=d,
            size=ws, o=out):
        return L.cmolhip_attn_window(c, n, p(q), p(k), p(v), p(slots), stride, p(lens), heads, kv, dh, ctx_, 0, win_, sinks,
                                     p(ws_), size, p(o))

    def pro(c=ctx.h, n=2, pos=0, q=d, k=d, v=d, heads=4, kv=2, dh=64, ctx_=8, win_=4, sinks=1, ws_=d, size=ws, o=out):
        return L.cmolhip_attn_window_prompt(c, n, pos, p(q), p(k), p(v), heads, kv, dh, ctx_, 0, win_, sinks, p(ws_), size, p(o))

    def sha(c=ctx.h, n=1, q=d, pk=d, pv=d, pre=4, pctx=4, k=d, v=d, stride=0, lens=d, heads=4, kv=2, dh=64, ctx_=8, ws_=d,
            size=ws, o=out):
        return L.cmolhip_attn_shared(c, n, p(q), p(pk), p(pv), pre, pctx, p(k), p(v), None, stride, p(lens), heads, kv, dh,
                                     ctx_, 0, p(ws_), size, p(o))

    for f in (win, pro, sha):
        for bad in (dict(c=None), dict(n=0), dict(n=65536), dict(q=None), dict(k=None), dict(v=None), dict(o=None),
                    dict(heads=3), dict(kv=0), dict(ctx_=0), dict(ctx_=(1 << 30) + 1), dict(ws_=None), dict(size=0), dict(q=d + 4), dict(k=d + 2),
                    dict(v=d + 8), dict(ws_=d + 4), dict(o=out + 4)):
            assert f(**bad) == A, (f.__name__, bad)
        assert f(dh=48) == native.CMOL_ERR_UNSUPPORTED
    for f in (win, sha):
        for bad in (dict(lens=None), dict(stride=8), dict(stride=2 * 8 * 64 + 4)):
            assert f(**bad) == A, (f.__name__, bad)
    for f in (win, pro):
        for bad in (dict(win_=0), dict(win_=-1), dict(sinks=-1)):
            assert f(**bad) == A, (f.__name__, bad)
    for bad in (dict(pos=-1), dict(pos=7), dict(n=9), dict(pos=2**31 - 1)):
        assert pro(**bad) == A, bad
    for bad in (dict(pre=-1), dict(pre=5), dict(pk=None), dict(pv=None), dict(pk=d + 8), dict(pctx=3)):
        assert sha(**bad) == A, bad

    def lg(size=ws, ws_=d, **kw):
        t = native.Logits()
        t.n, t.vocab, t.stride, t.logits, t.out, t.next = 1, 16, 16, d, out, None
        for a, b in kw.items():
            setattr(t, a, b)
        return L.cmolhip_logits(ctx.h, C.byref(t), p(ws_), size)

    for bad in (dict(n=0), dict(n=65536), dict(vocab=0), dict(stride=15), dict(logits=None), dict(out=None), dict(size=0),
                dict(ws_=None), dict(ws_=d + 8), dict(history=d), dict(history=d, history_len=d, history_cap=-1),
                dict(bias_ids=d), dict(bias_ids=d, bias=d), dict(bias_ids=d, bias=d, bias_len=d, bias_cap=-1),
                dict(mask=d), dict(mask=d, mask_rows=0, mask_row=d), dict(mask=d, mask_rows=1, n=2)):
        assert lg(**bad) == A, bad
    native.check(L.cmolhip_synchronize(ctx.h), "sync")
    assert np.all(ctx.d2h(out, 1024, np.float32) == 5.0)


def serving_step(ctx, seed, n=4):
    """Windowed attention, attention behind a prefix and the choice of a token,
    as one step of a server: the calls (to run any number of times), and a
    check of their outputs."""
    L = native.lib()
    heads, kv, dh, max_ctx, window, sinks, prefix, V = 16, 4, 128, 700, 200, 4, 500, 5000
    rng = np.random.default_rng(seed)
    q = rng.standard_normal((n, heads, dh)).astype(np.float32)
    k, v = (rand_cache(rng, (n, kv, max_ctx, dh), 1) for _ in range(2))
    pk, pv = (rand_cache(rng, (kv, prefix, dh), 1) for _ in range(2))
    lens = [int(t) for t in rng.integers(1, max_ctx, n)]
    x = rng.standard_normal((n, V)).astype(np.float32)
    dq, dk, dv, dpk, dpv, dx = (ctx.upload(a) for a in (q, k, v, pk, pv, x))
    dl = ctx.upload(np.array(lens, np.int32))
    dr = ctx.upload(np.full(n, 1.1, np.float32))
    hist = rng.integers(0, V, (n, 64)).astype(np.int32)
    dh_, dhl = ctx.upload(hist), ctx.upload(np.full(n, 64, np.int32))
    o1, o2, o3, nx = ctx.alloc(q.nbytes), ctx.alloc(q.nbytes), ctx.alloc(x.nbytes), ctx.alloc(4 * n)
    b = [L.cmolhip_attn_window_bytes(n, heads, kv, dh, max_ctx, window, sinks),
         L.cmolhip_attn_shared_bytes(n, heads, kv, dh, prefix, max_ctx), L.cmolhip_logits_bytes(n, V)]
    ws = ctx.alloc(max(b))
    t = native.Logits()
    t.n, t.vocab, t.stride, t.logits, t.out, t.next = n, V, V, dx, o3, nx
    t.history, t.history_len, t.history_cap, t.repeat = dh_, dhl, 64, dr

    def calls(c=None):
        h = (c or ctx).h
        native.check(L.cmolhip_attn_window(h, n, p(dq), p(dk), p(dv), None, 0, p(dl), heads, kv, dh, max_ctx, 1, window,
                                           sinks, p(ws), b[0], p(o1)))
        native.check(L.cmolhip_attn_shared(h, n, p(dq), p(dpk), p(dpv), prefix, prefix, p(dk), p(dv), None, 0, p(dl), heads,
                                           kv, dh, max_ctx, 1, p(ws), b[1], p(o2)))
        native.check(L.cmolhip_logits(h, C.byref(t), p(ws), b[2]))

    wants = []
    for i in range(n):
        a = reference(q[i].astype(np.float64), k[i].astype(np.float64), v[i].astype(np.float64),
                      window_seen(lens[i], max_ctx, window, sinks))
        kk = np.concatenate([pk, k[i][:, :lens[i]]], 1).astype(np.float64)
        vv = np.concatenate([pv, v[i][:, :lens[i]]], 1).astype(np.float64)
        wants.append((a, reference(q[i].astype(np.float64), kk, vv, np.ones(kk.shape[1], bool)),
                      logits_reference(x[i], hist[i], np.float32(1.1), 0, 0, [], None)))

    def check(what):
        g1, g2 = (ctx.d2h(o, (n, heads, dh), np.float32) for o in (o1, o2))
        g3, gn = ctx.d2h(o3, (n, V), np.float32), ctx.d2h(nx, n, np.int32)
        for i, (a, s, l) in enumerate(wants):
            close(g1[i], *a, f"{what}: window {i}")
            close(g2[i], *s, f"{what}: shared {i}")
            assert np.array_equal(g3[i], l[0]) and gn[i] == l[1], f"{what}: logits {i}"
        for o in (o1, o2, o3, nx):
            ctx.h2d(o, np.full(n, np.nan, np.float32))

    return calls, check


def test_a_step_of_a_server(ctx):
    calls, check = serving_step(ctx, 1)
    for _ in range(2):
        calls()
        native.check(native.lib().cmolhip_synchronize(ctx.h))
        check("eager")


def test_captured_steps(ctx):
    """Two steps captured into graphs with a workspace each, replayed several
    times with eager work between; the second graph runs on another stream."""
    rt = hiprt.rt()
    stream = C.c_void_p(native.lib().cmolhip_stream(ctx.h))
    steps = [serving_step(ctx, 2), serving_step(ctx, 3, n=7)]
    execs = []
    for calls, _ in steps:
        graph, ex = C.c_void_p(), C.c_void_p()
        assert rt.hipStreamBeginCapture(stream, 1) == 0   # thread-local mode
        calls()
        assert rt.hipStreamEndCapture(stream, C.byref(graph)) == 0
        assert rt.hipGraphInstantiate(C.byref(ex), graph, None, None, C.c_size_t(0)) == 0
        execs.append((graph, ex))
    other = native.Ctx(0)
    streams = [stream, C.c_void_p(native.lib().cmolhip_stream(other.h))]
    eager, check_eager = serving_step(ctx, 4)
    for turn in range(3):
        for (_, ex), s in zip(execs, streams):
            assert rt.hipGraphLaunch(ex, s) == 0
        eager()
        hiprt.device_synchronize()
        for i, (_, check) in enumerate(steps):
            check(f"replay {turn} of graph {i}")
        check_eager(f"beside replay {turn}")
    for graph, ex in execs:
        rt.hipGraphExecDestroy(ex)
        rt.hipGraphDestroy(graph)
    other.close()


@pytest.mark.parametrize("form", ["0", "1"])
@pytest.mark.parametrize("f16", [F32, F16])
def test_captured_prompts(ctx, monkeypatch, f16, form):
    """A prompt in both of its forms captured into a graph and replayed over
    other queries and another cache in the same places, with an eager prompt
    between; its result is the eager call's, bit for bit."""
    prompt_form(monkeypatch, form)
    rt, L = hiprt.rt(), native.lib()
    stream = C.c_void_p(L.cmolhip_stream(ctx.h))
    heads, kv, dh, n, pos0, max_ctx, window, sinks = 16, 4, 128, 70, 300, 400, 150, 4
    rng = np.random.default_rng(12)
    need = L.cmolhip_attn_window_prompt_bytes(n, heads, kv, dh, max_ctx, window, sinks)
    size = kv * max_ctx * dh * (2 if f16 else 4)
    ws, out, dq, dk, dv = ctx.alloc(need), ctx.alloc(n * heads * dh * 4), ctx.alloc(n * heads * dh * 4), ctx.alloc(size), ctx.alloc(size)
    graph, ex = C.c_void_p(), C.c_void_p()
    assert rt.hipStreamBeginCapture(stream, 1) == 0   # thread-local mode
    native.check(L.cmolhip_attn_window_prompt(ctx.h, n, pos0, p(dq), p(dk), p(dv), heads, kv, dh, max_ctx, f16, window, sinks,
                                              p(ws), need, p(out)))
    assert rt.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert rt.hipGraphInstantiate(C.byref(ex), graph, None, None, C.c_size_t(0)) == 0
    for turn in range(3):
        q = rng.standard_normal((n, heads, dh)).astype(np.float32)
        k, v = (rand_cache(rng, (kv, max_ctx, dh), f16) for _ in range(2))
        for d, x in ((dq, q), (dk, k), (dv, v), (out, np.full(n * heads * dh, 777.0, np.float32))):
            ctx.h2d(d, x)
        assert rt.hipGraphLaunch(ex, stream) == 0
        native.check(L.cmolhip_synchronize(ctx.h))
        got = ctx.d2h(out, (n, heads, dh), np.float32)
        eager = prompt_call(ctx, q, ctx.upload(k), ctx.upload(v), pos0, heads, kv, dh, max_ctx, f16, window, sinks)
        assert np.array_equal(got, eager), f"replay {turn}"
        want, tol = reference(q[-1].astype(np.float64), k.astype(np.float64), v.astype(np.float64),
                              window_seen(pos0 + n, max_ctx, window, sinks))
        close(got[-1], want, tol, f"replay {turn}")
    rt.hipGraphExecDestroy(ex)
    rt.hipGraphDestroy(graph)


def test_equal_calls_give_equal_bits(ctx):
    """The same call twice, its scratch full of something else: no order of work
    reaches the result."""
    heads, kv, dh, max_ctx = 8, 2, 128, 1500
    rng = np.random.default_rng(13)
    for f16 in (F32, F16):
        q = rng.standard_normal((5, heads, dh)).astype(np.float32)
        k, v = (rand_cache(rng, (5, kv, max_ctx, dh), f16) for _ in range(2))
        dk, dv = ctx.upload(k), ctx.upload(v)
        lens = [1500, 3, 700, 0, 64]
        a = [window_call(ctx, q, dk, dv, None, 0, lens, heads, kv, dh, max_ctx, f16, 1300, 4) for _ in range(2)]
        assert np.array_equal(*a)
        a = [shared_call(ctx, q, dk, dv, 1200, max_ctx, dk, dv, None, 0, lens, heads, kv, dh, max_ctx, f16) for _ in range(2)]
        assert np.array_equal(*a)


def test_steps_of_two_threads(ctx):
    """Calls of two threads on one context and of a third on its own, each with
    its workspace."""
    other = native.Ctx(0)
    steps = [serving_step(ctx, s) for s in (5, 6, 7)]
    errors = []

    def work(calls, c):
        try:
            for _ in range(20):
                calls(c)
        except Exception as e:   # noqa: BLE001
            errors.append(e)

    ts = [threading.Thread(target=work, args=(s[0], c)) for s, c in zip(steps, (ctx, ctx, other))]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    hiprt.device_synchronize()
    assert not errors
    for i, s in enumerate(steps):
        s[1](f"thread {i}")
    other.close()


@pytest.mark.parametrize("form", [None, "0", "1"])
@pytest.mark.parametrize("f16", [F32, F16])
def test_as_many_rows_as_a_call_takes(ctx, monkeypatch, f16, form):
    """65535 sessions, tokens and rows of logits."""
    session_form(monkeypatch, form)
    prompt_form(monkeypatch, form)
    c = native.Ctx(512 << 20)
    n, heads, kv, dh, max_ctx, prefix = 65535, 2, 1, 64, 3, 2
    rng = np.random.default_rng(14)
    q = rng.standard_normal((n, heads, dh)).astype(np.float32)
    k, v = (rand_cache(rng, (100, kv, max_ctx, dh), f16) for _ in range(2))
    slots, lens = rng.integers(-1, 100, n).astype(np.int32), rng.integers(-1, max_ctx + 2, n).astype(np.int32)
    dk, dv = c.upload(k), c.upload(v)
    win = window_call(c, q, dk, dv, slots, 0, lens, heads, kv, dh, max_ctx, f16, 2, 0)
    sha = shared_call(c, q, dk, dv, prefix, max_ctx, dk, dv, slots, 0, lens, heads, kv, dh, max_ctx, f16)
    long_k, long_v = (rand_cache(rng, (kv, n, dh), f16) for _ in range(2))
    pro = prompt_call(c, q, c.upload(long_k), c.upload(long_v), 0, heads, kv, dh, n, f16, 40, 1)
    k64, v64 = k.astype(np.float64), v.astype(np.float64)
    for i in [0, 1, n - 2, n - 1] + [int(t) for t in rng.integers(0, n, 60)]:
        m = 0 if slots[i] < 0 else max(0, min(lens[i], max_ctx))
        qi = q[i].astype(np.float64)
        close(win[i], *reference(qi, k64[slots[i]], v64[slots[i]], window_seen(m, max_ctx, 2, 0)), f"session {i}")
        kk, vv = (np.concatenate([x[0][:, :prefix], x[slots[i]][:, :m]], 1) for x in (k64, v64))
        close(sha[i], *reference(qi, kk, vv, np.ones(prefix + m, bool)), f"session {i} behind the prefix")
        t = np.unique(np.concatenate([[0], np.arange(max(0, i - 39), i + 1)]))
        close(pro[i], *reference(qi, long_k[:, t].astype(np.float64), long_v[:, t].astype(np.float64), np.ones(len(t), bool)),
              f"token {i}")
    c.close()
    x = rng.standard_normal((n, 40)).astype(np.float32)
    got, nxt = logits_call(ctx, x)
    assert np.array_equal(got, x) and np.array_equal(nxt, x.argmax(1))


@pytest.mark.parametrize("f16", [F32, F16])
def test_offsets_past_32_bits(gpu, f16):
    """A cache whose positions lie more than 4 GiB from its start; only the
    positions that are seen are written."""
    heads, kv, dh, window, sinks = 4, 2, 16, 70, 3
    es = 2 if f16 else 4
    max_ctx = (1 << 32) // (dh * es) + 1000
    size = kv * max_ctx * dh * es
    c = gpu.Ctx(2 * size + (64 << 20))
    dk, dv = c.alloc(size), c.alloc(size)
    rng = np.random.default_rng(6)
    L = max_ctx - 5
    kk, vv = (rand_cache(rng, (kv, sinks + window, dh), f16) for _ in range(2))
    for d, a in ((dk, kk), (dv, vv)):
        for h in range(kv):
            c.h2d(d + h * max_ctx * dh * es, a[h, :sinks])
            c.h2d(d + (h * max_ctx + L - window) * dh * es, a[h, sinks:])
    q = rng.standard_normal((1, heads, dh)).astype(np.float32)
    want, tol = reference(q[0].astype(np.float64), kk.astype(np.float64), vv.astype(np.float64), np.ones(sinks + window, bool))
    got = window_call(c, q, dk, dv, None, 0, [L], heads, kv, dh, max_ctx, f16, window, sinks)
    close(got[0], want, tol, "window")
    got = prompt_call(c, q, dk, dv, L - 1, heads, kv, dh, max_ctx, f16, window, sinks)
    close(got[0], want, tol, "prompt")
    # the last window positions as the second kv head's shared prefix, far from its start
    got = shared_call(c, q, dk + (L - window) * dh * es, dv + (L - window) * dh * es, window, max_ctx, dk, dv, None, 0,
                      [sinks], heads, kv, dh, max_ctx, f16)
    close(got[0], want, tol, "shared")
    c.close()
