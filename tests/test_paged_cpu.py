"""The paged calls refuse what they cannot do before anything is launched (no device needed)."""
import ctypes as C

import pytest

from tinycoder_inference_b200 import capi

lib = capi.lib
P = 1 << 20   # a fake, aligned address: every check below fails before anything is dereferenced or launched


def cache(**kw):
    c = capi.PagedKv()
    for f in ("k", "v", "ks", "vs", "pages", "lens"):
        setattr(c, f, P)
    c.batch, c.pagesPerSeq, c.numPages, c.pageRows, c.nKV, c.hd, c.tokens, c.kvI8 = 2, 8, 64, 16, 4, 128, 2, 1
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def write(c, k=P, v=P, q=None, q_out=None, half=0, heads=0, cos=None, sin=None, rows=0):
    return lib.tc_paged_kv_write(C.byref(c), k, v, q, q_out, half, heads, cos, sin, rows, None)


def read(c, k=P, v=P, half=0):
    return lib.tc_paged_kv_read(C.byref(c), k, v, half, None)


def workspace():
    n = C.c_size_t()
    assert lib.tc_attn_paged_workspace_bytes(C.byref(n)) == 0
    return n.value


def attend(c, q=P, out=P, half=0, heads=28, most=1, scale=0.1, ws=P, size=None):
    return lib.tc_attn_paged(C.byref(c), q, out, half, heads, most, scale, ws, workspace() if size is None else size, None)


BAD_CACHES = [
    (dict(k=None), capi.TC_EINVAL), (dict(v=None), capi.TC_EINVAL), (dict(pages=None), capi.TC_EINVAL),
    (dict(lens=None), capi.TC_EINVAL), (dict(ks=None), capi.TC_EINVAL), (dict(vs=None), capi.TC_EINVAL),
    (dict(batch=0), capi.TC_EINVAL), (dict(pagesPerSeq=0), capi.TC_EINVAL), (dict(numPages=0), capi.TC_EINVAL),
    (dict(pageRows=0), capi.TC_EINVAL), (dict(nKV=0), capi.TC_EINVAL), (dict(k=P + 8), capi.TC_EINVAL),
    (dict(hd=64), capi.TC_EUNSUPPORTED), (dict(hd=96), capi.TC_EUNSUPPORTED), (dict(hd=512, kvI8=0), capi.TC_EUNSUPPORTED),
    (dict(pageRows=12), capi.TC_EUNSUPPORTED), (dict(pageRows=1), capi.TC_EUNSUPPORTED),
    (dict(tokens=3), capi.TC_EINVAL),                         # three tokens of two sequences need `starts`
    (dict(pagesPerSeq=1 << 30, pageRows=1 << 10), capi.TC_EUNSUPPORTED), (dict(numPages=1 << 31), capi.TC_EUNSUPPORTED),
]


@pytest.mark.parametrize("change, code", BAD_CACHES, ids=[str(c) for c, _ in BAD_CACHES])
def test_every_paged_call_checks_the_cache(change, code):
    for call in (write, read, attend):
        assert call(cache(**change)) == code
        assert lib.tc_last_error()


def test_null_descriptors():
    assert lib.tc_paged_kv_write(None, P, P, None, None, 0, 0, None, None, 0, None) == capi.TC_EINVAL
    assert lib.tc_paged_kv_read(None, P, P, 0, None) == capi.TC_EINVAL
    assert lib.tc_attn_paged(None, P, P, 0, 28, 1, 0.1, P, 1 << 30, None) == capi.TC_EINVAL
    assert lib.tc_attn_paged_workspace_bytes(None) == capi.TC_EINVAL


def test_write_refusals():
    c = cache()
    assert write(c, k=None) == capi.TC_EINVAL
    assert write(c, cos=P, rows=5) == capi.TC_EINVAL                                # one table
    assert write(c, q=P, heads=28) == capi.TC_EINVAL                               # q without a place
    assert write(c, q=P, q_out=P, heads=0) == capi.TC_EINVAL
    assert write(c, q=P, q_out=P, half=1, heads=28) == capi.TC_EINVAL and b"in place" in lib.tc_last_error()
    assert write(c, k=P + 4) == capi.TC_EINVAL and b"alignment" in lib.tc_last_error()
    assert write(c, q=P, q_out=P + 8, heads=28) == capi.TC_EINVAL
    assert write(cache(tokens=0), k=None, v=None) == 0                              # nothing to do


def test_read_refusals():
    assert read(cache(), k=None) == capi.TC_EINVAL
    assert read(cache(), v=P + 2) == capi.TC_EINVAL
    assert read(cache(tokens=0), k=None, v=None) == 0


def test_attention_refusals():
    c = cache()
    assert attend(c, heads=0) == capi.TC_EINVAL
    assert attend(c, heads=30) == capi.TC_EINVAL                                    # 30 heads over 4
    assert attend(c, heads=4 * 129) == capi.TC_EUNSUPPORTED
    assert attend(cache(tokens=1 << 30), heads=28) == capi.TC_EUNSUPPORTED          # 2^30 tokens of 28 heads
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        assert attend(c, scale=scale) == capi.TC_EINVAL
    for null in ("q", "out", "ws"):
        assert attend(c, **{null: None}) == capi.TC_EINVAL
    assert attend(c, q=P + 8) == capi.TC_EINVAL
    assert attend(c, size=workspace() - 1) == capi.TC_EWORKSPACE
    assert attend(cache(tokens=0), q=None, out=None, ws=None) == 0
