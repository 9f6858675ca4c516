"""What the serving operators (include/cmol_hip.h) refuse, without a device:
their workspace sizes, which are 0 for arguments that the calls refuse, and the
calls themselves without a context."""
import ctypes as C

import pytest

from libcmol_amd import native

INT_MAX = 2**31 - 1


def window(n=2, heads=4, kv=2, dh=64, ctx=100, window=16, sinks=2):
    return n, heads, kv, dh, ctx, window, sinks


BAD_SHAPES = [dict(n=0), dict(n=-1), dict(n=65536), dict(heads=0), dict(heads=3), dict(heads=1), dict(kv=0), dict(kv=-2),
              dict(dh=0), dict(dh=-64), dict(dh=48), dict(dh=8), dict(dh=512), dict(ctx=0), dict(ctx=-5), dict(ctx=(1 << 30) + 1),
              dict(n=65535, heads=256)]


@pytest.mark.parametrize("bad", BAD_SHAPES + [dict(window=0), dict(window=-1), dict(sinks=-1)], ids=str)
@pytest.mark.parametrize("name", ["cmolhip_attn_window_bytes", "cmolhip_attn_window_prompt_bytes"])
def test_window_bytes_refuse(name, bad):
    f = getattr(native.lib(), name)
    assert f(*window()) > 0
    assert f(*window(**bad)) == 0


@pytest.mark.parametrize("bad", BAD_SHAPES, ids=str)
def test_shared_bytes_refuse(bad):
    f = native.lib().cmolhip_attn_shared_bytes
    args = dict(n=2, heads=4, kv=2, dh=64, prefix=100, ctx=100)
    assert f(*args.values()) > 0
    assert f(*{**args, **bad}.values()) == 0
    assert f(2, 4, 2, 64, -1, 100) == 0
    assert f(2, 4, 2, 64, (1 << 30) + 1, 100) == 0
    assert f(2, 4, 2, 64, 0, 100) > 0


def test_prompt_bytes_refuse_tokens_past_the_cache():
    f = native.lib().cmolhip_attn_window_prompt_bytes
    assert f(*window(n=100)) > 0
    assert f(*window(n=101)) == 0


def test_bytes_refuse_more_kv_heads_than_a_grid_holds():
    L = native.lib()
    for kv, takes in ((65535, True), (65536, False)):
        assert (L.cmolhip_attn_window_bytes(1, kv, kv, 16, 1, 1, 0) > 0) == takes
        assert (L.cmolhip_attn_window_prompt_bytes(1, kv, kv, 64, 1, 1, 0) > 0) == takes
        assert (L.cmolhip_attn_shared_bytes(1, kv, kv, 16, 1, 1) > 0) == takes


def test_bytes_at_the_largest_arguments():
    """Sizes that pass 32 bits come out whole; a window or a sink count past
    the cache is the cache's length."""
    L = native.lib()
    for heads, kv, dh in ((1, 1, 16), (16, 4, 128), (32, 1, 256)):
        one = L.cmolhip_attn_window_bytes(1, heads, kv, dh, 4096, INT_MAX, INT_MAX)
        assert one == L.cmolhip_attn_window_bytes(1, heads, kv, dh, 4096, 4096, 4096)
        # (not more for more sessions: those that fill the chip each have one work-group and no partial results)
        assert 0 < L.cmolhip_attn_window_bytes(65535, heads, kv, dh, 1 << 20, INT_MAX, INT_MAX) < 1 << 46
        assert 0 < L.cmolhip_attn_shared_bytes(65535, heads, kv, dh, 1 << 20, 1 << 20) < 1 << 46
        assert 0 < L.cmolhip_attn_window_prompt_bytes(65535, heads, kv, dh, 1 << 20, INT_MAX, 0) < 1 << 46
    assert L.cmolhip_logits_bytes(1, 1) > 0
    assert L.cmolhip_logits_bytes(65535, INT_MAX) > 0
    for n, v in ((0, 100), (-1, 100), (65536, 100), (1, 0), (1, -7)):
        assert L.cmolhip_logits_bytes(n, v) == 0


def test_calls_without_a_context():
    L = native.lib()
    p = C.c_void_p(4096)
    assert L.cmolhip_attn_window(None, 2, p, p, p, None, 0, p, 4, 2, 64, 100, 0, 16, 2, p, 1 << 20, p) == native.CMOL_ERR_ARGS
    assert L.cmolhip_attn_window_prompt(None, 2, 0, p, p, p, 4, 2, 64, 100, 0, 16, 2, p, 1 << 20, p) == native.CMOL_ERR_ARGS
    assert L.cmolhip_attn_shared(None, 2, p, p, p, 8, 8, p, p, None, 0, p, 4, 2, 64, 100, 0, p, 1 << 20,
                                 p) == native.CMOL_ERR_ARGS
    assert L.cmolhip_attn_window(None, 2, p, p, p, None, 0, p, 4, 2, 48, 100, 0, 16, 2, p, 1 << 20,
                                 p) == native.CMOL_ERR_UNSUPPORTED
    d = native.Logits()
    assert L.cmolhip_logits(None, C.byref(d), p, 1 << 20) == native.CMOL_ERR_ARGS
    assert L.cmolhip_logits(None, None, p, 1 << 20) == native.CMOL_ERR_ARGS
