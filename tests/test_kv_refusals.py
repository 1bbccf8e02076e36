"""What the paged key-value cache's operators refuse, without a GPU: the library's
entry points check their arguments before they look at the device, the wrappers
before they call the library."""

from __future__ import annotations

import ctypes

import pytest
import torch

from uma_qmoe_amd import _native
from uma_qmoe_amd.native_backend import HipExtension, KVCache

A, B, C, D, E, F, G = (i << 24 for i in range(1, 8))  # addresses that nothing reads


@pytest.fixture(scope="module")
def lib():
    return _native.library()


def cache(key=A, value=B, ks=None, vs=None, pages=4, kv_heads=2, page_size=16, head_dim=64):
    return _native.KVCache(key, value, ks, vs, pages, kv_heads, page_size, head_dim)


BAD_CACHES = [
    (dict(key=None), "required"), (dict(value=None), "required"), (dict(ks=C), "together"), (dict(vs=C), "together"),
    (dict(key=A + 8), "aligned"), (dict(value=B + 4), "aligned"), (dict(ks=C + 4, vs=D), "aligned"), (dict(ks=C, vs=D + 8), "aligned"),
    (dict(pages=0), "pages"), (dict(pages=-1), "pages"), (dict(pages=1 << 31), "pages"),
    (dict(pages=(1 << 31) - 1, kv_heads=65535, head_dim=256), "2^48"),
    (dict(kv_heads=0), "kv_heads"), (dict(kv_heads=65536), "kv_heads"), (dict(kv_heads=-1), "kv_heads"),
    (dict(page_size=0), "page_size"), (dict(page_size=8), "page_size"), (dict(page_size=48), "page_size"),
    (dict(page_size=512), "page_size"), (dict(page_size=-16), "page_size"),
    (dict(head_dim=0), "head_dim"), (dict(head_dim=8), "head_dim"), (dict(head_dim=72), "head_dim"),
    (dict(head_dim=272), "head_dim"), (dict(head_dim=-16), "head_dim"),
]

APPEND = dict(key=C, kb=1280, kh=640, kt=64, value=D, vb=1280, vh=640, vt=64, batch=3, tokens=10, table=E, stride=4, width=4,
              starts=F, counts=G)
READ = dict(batch=3, table=E, stride=4, width=4, lengths=F, most=50, key=C, value=D)
ATTEND = dict(query=C, batch=3, heads=4, table=E, stride=4, width=4, lengths=F, scale=0.125, window=0, out=D, ws=G, bytes=1 << 23)
CALLS = {"uqm_kv_append": APPEND, "uqm_kv_read": READ, "uqm_paged_attention": ATTEND}


def refused(lib, name, kv, words, code=1, **changed):
    args = {**CALLS[name], **changed}
    rc = getattr(lib, name)(None if kv is None else ctypes.byref(kv), *args.values(), None)
    message = lib.uqm_last_error().decode()
    assert rc == code, (rc, message)
    assert words in message, message


@pytest.mark.parametrize("name", CALLS)
def test_caches(lib, name):
    refused(lib, name, None, "a cache is required")
    for changed, words in BAD_CACHES:
        refused(lib, name, cache(**changed), words)


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("changed,words", [
    (dict(batch=-1), "batch"), (dict(batch=1 << 31), "batch"), (dict(width=-1), "max_pages"),
    (dict(width=(1 << 26) + 1, stride=1 << 27), "max_pages"), (dict(stride=3), "table_stride"), (dict(stride=1 << 31), "table_stride"),
    (dict(stride=1 << 30, batch=1 << 20), "2^48"), (dict(table=None), "required"), (dict(table=E + 2), "aligned"),
])
def test_tables(lib, name, changed, words):
    refused(lib, name, cache(), words, **changed)


@pytest.mark.parametrize("changed,words", [
    (dict(tokens=-1), "tokens"), (dict(tokens=1 << 30), "tokens"),
    (dict(key=None), "required"), (dict(value=None), "required"), (dict(starts=None), "required"),
    (dict(key=C + 8), "aligned"), (dict(value=D + 2), "aligned"), (dict(starts=F + 1), "aligned"), (dict(counts=G + 2), "aligned"),
    (dict(kb=-8), "strides"), (dict(kh=4), "strides"), (dict(kt=1), "strides"), (dict(vb=1 << 50), "strides"),
    (dict(vh=-64), "strides"), (dict(vt=63), "strides"),
    (dict(key=A - 16), "overlaps an input"), (dict(value=B + 4096), "overlaps an input"), (dict(table=A), "overlaps an input"),
    (dict(starts=B), "overlaps an input"), (dict(counts=A + 16380), "overlaps an input"),
])
def test_append(lib, changed, words):
    refused(lib, "uqm_kv_append", cache(), words, **changed)


@pytest.mark.parametrize("kv", [
    dict(value=A), dict(value=A + 16), dict(ks=E, vs=E), dict(ks=E, vs=E + 256), dict(ks=A, vs=E), dict(ks=E, vs=B), dict(ks=B, vs=E),
    dict(ks=E, vs=A + 4096)])
def test_append_keeps_the_parts_apart(lib, kv):
    refused(lib, "uqm_kv_append", cache(**kv), "two parts of the cache overlap", table=F + 65536)


@pytest.mark.parametrize("changed,words", [
    (dict(most=-1), "max_length"), (dict(most=1 << 30), "max_length"), (dict(batch=1 << 30, most=1 << 29, stride=4), "max_length"),
    (dict(lengths=None), "required"), (dict(key=None), "required"), (dict(value=None), "required"),
    (dict(key=C + 8), "aligned"), (dict(value=D + 2), "aligned"), (dict(lengths=F + 2), "aligned"),
    (dict(key=A + 16), "overlaps an input"), (dict(value=B - 16), "overlaps an input"), (dict(key=E - 16), "overlaps an input"),
    (dict(value=F), "overlaps an input"), (dict(key=D + 16), "two outputs overlap"),
])
def test_read(lib, changed, words):
    refused(lib, "uqm_kv_read", cache(), words, **changed)


@pytest.mark.parametrize("changed,words", [
    (dict(heads=0), "multiple"), (dict(heads=3), "multiple"), (dict(heads=-2), "multiple"), (dict(heads=1 << 24), "2^24"),
    (dict(batch=1 << 20, heads=16), "2^24"),
    (dict(batch=1 << 6, heads=2, width=1 << 26, stride=1 << 26), "room"), (dict(scale=float("nan")), "finite"), (dict(scale=float("inf")), "finite"),
    (dict(window=-1), "window"), (dict(query=None), "required"), (dict(lengths=None), "required"), (dict(out=None), "required"),
    (dict(query=C + 8), "aligned"), (dict(out=D + 2), "aligned"), (dict(lengths=F + 3), "aligned"),
    (dict(out=C + 16), "overlaps"), (dict(out=A), "overlaps"), (dict(out=E), "overlaps"), (dict(out=F), "overlaps"),
])
def test_attention(lib, changed, words):
    refused(lib, "uqm_paged_attention", cache(), words, **changed)


def test_no_work(lib):
    kv = ctypes.byref(cache())
    for name, changed in (("uqm_kv_append", dict(batch=0)), ("uqm_kv_append", dict(tokens=0)), ("uqm_kv_append", dict(width=0)),
                          ("uqm_kv_read", dict(batch=0)), ("uqm_kv_read", dict(most=0)), ("uqm_paged_attention", dict(batch=0))):
        args = {**CALLS[name], **changed}
        assert getattr(lib, name)(kv, *(None if k in ("key", "value", "query", "table", "starts", "lengths", "out", "ws") else v
                                        for k, v in args.items()), None) == 0, (name, changed)


def test_workspace_of_refused_sizes(lib):
    good = (3, 4, 2, 64, 16, 400, 0)
    assert lib.uqm_paged_attention_workspace_bytes(*good) > 0
    for i, bad in enumerate((-1, 3, 0, 60, 15, -1, -1)):
        sizes = (*good[:i], bad, *good[i + 1:])
        assert lib.uqm_paged_attention_workspace_bytes(*sizes) == 0


# ---------------------------------------------------------------- wrappers --
@pytest.fixture(scope="module")
def ext():
    return HipExtension()


def bf(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def kv(dtype=torch.bfloat16, shape=(4, 2, 16, 64), scales=None):
    data = [torch.zeros(shape, dtype=torch.uint8).view(dtype) if dtype is torch.float8_e4m3fn else torch.zeros(shape, dtype=dtype)
            for _ in range(2)]
    return KVCache(*data, *(scales or (None, None)))


F8 = torch.float8_e4m3fn
GOOD_SCALES = (torch.zeros(4, 2, 16), torch.zeros(4, 2, 16))


@pytest.mark.parametrize("bad,words", [
    (KVCache(bf(4, 2, 16, 64), bf(4, 2, 16, 32)), "one shape"),
    (KVCache(bf(4, 2, 16), bf(4, 2, 16)), "one shape"),
    (KVCache(bf(4, 2, 16, 64), torch.zeros(4, 2, 16, 64)), "one shape and type"),
    (kv(torch.float32), "BF16 or float8"),
    (kv(F8), "scales with a float8"),
    (kv(F8, scales=(GOOD_SCALES[0], None)), "scales with a float8"),
    (kv(scales=GOOD_SCALES), "scales with a float8"),
    (kv(F8, scales=(torch.zeros(4, 2, 8), torch.zeros(4, 2, 8))), "float32 scales"),
    (kv(F8, scales=(GOOD_SCALES[0].double(), GOOD_SCALES[1])), "float32 scales"),
    (KVCache(bf(4, 2, 64, 16).transpose(2, 3), bf(4, 2, 64, 16).transpose(2, 3)), "contiguous"),
    (kv(), "device"),
    (kv(F8, scales=GOOD_SCALES), "device"),
])
def test_wrappers_look_at_the_cache(ext, bad, words):
    for call in (lambda: ext.kv_append(bad, bf(1, 2, 3, 64), bf(1, 2, 3, 64), i32(1, 4), i32(1)),
                 lambda: ext.kv_read(bad, i32(1, 4), i32(1), 5),
                 lambda: ext.paged_attention(bf(1, 2, 64), bad, i32(1, 4), i32(1))):
        with pytest.raises(RuntimeError, match=words):
            call()


@pytest.mark.parametrize("args", [(0, 2, 16, 64), (4, 0, 16, 64), (4, 2, 24, 64), (4, 2, 512, 64), (4, 2, 16, 0), (4, 2, 16, 72), (4, 2, 16, 272)])
def test_new_cache(ext, args):
    with pytest.raises(RuntimeError, match="new_kv_cache requires"):
        ext.new_kv_cache(*args, device="cpu")


def test_new_cache_is_zeros(ext):
    a, b = ext.new_kv_cache(3, 2, 16, 32, device="cpu"), ext.new_kv_cache(3, 2, 16, 32, fp8=True, device="cpu")
    assert a.key.shape == b.key.shape == (3, 2, 16, 32) and a.key_scales is None and a.key.dtype is torch.bfloat16
    assert b.key.dtype is F8 and b.value_scales.shape == (3, 2, 16) and not b.value.float().any()


class OnDevice0:
    """A CPU tensor that says it is on device 0, so that checks behind the device's are reached here."""

    def __init__(self, t):
        self.t = t

    def get_device(self):
        return 0

    def __getattr__(self, name):
        return getattr(self.t, name)


def dev(t):
    return OnDevice0(t)


GOOD = KVCache(dev(bf(4, 2, 16, 64)), dev(bf(4, 2, 16, 64)))


@pytest.mark.parametrize("call,words", [
    (lambda e: e.kv_append(GOOD, dev(bf(1, 2, 64)), dev(bf(1, 2, 64)), dev(i32(1, 4)), dev(i32(1))), "BF16 keys and values"),
    (lambda e: e.kv_append(GOOD, dev(bf(1, 3, 5, 64)), dev(bf(1, 3, 5, 64)), dev(i32(1, 4)), dev(i32(1))), "BF16 keys and values"),
    (lambda e: e.kv_append(GOOD, dev(bf(1, 2, 5, 32)), dev(bf(1, 2, 5, 32)), dev(i32(1, 4)), dev(i32(1))), "BF16 keys and values"),
    (lambda e: e.kv_append(GOOD, dev(bf(1, 2, 5, 64).float()), dev(bf(1, 2, 5, 64)), dev(i32(1, 4)), dev(i32(1))), "BF16 keys and values"),
    (lambda e: e.kv_append(GOOD, dev(bf(1, 2, 5, 64)), dev(bf(1, 2, 6, 64)), dev(i32(1, 4)), dev(i32(1))), "one shape"),
    (lambda e: e.kv_append(GOOD, dev(bf(1, 2, 5, 64)), bf(1, 2, 5, 64), dev(i32(1, 4)), dev(i32(1))), "one device"),
    (lambda e: e.kv_append(GOOD, dev(bf(1, 2, 5, 64)), dev(bf(1, 2, 5, 64)), dev(i32(2, 4)), dev(i32(2))), "each sequence"),
    (lambda e: e.kv_append(GOOD, dev(bf(1, 2, 5, 64)), dev(bf(1, 2, 5, 64)), dev(i32(1, 4).long()), dev(i32(1))), "int32 page table"),
    (lambda e: e.kv_append(GOOD, dev(bf(1, 2, 5, 64)), dev(bf(1, 2, 5, 64)), dev(i32(1)), dev(i32(1))), "int32 page table"),
    (lambda e: e.kv_append(GOOD, dev(bf(1, 2, 5, 64)), dev(bf(1, 2, 5, 64)), dev(i32(1, 4)), dev(i32(2))), "int32 entry"),
    (lambda e: e.kv_append(GOOD, dev(bf(1, 2, 5, 64)), dev(bf(1, 2, 5, 64)), dev(i32(1, 4)), dev(i32(1).long())), "int32 entry"),
    (lambda e: e.kv_append(GOOD, dev(bf(1, 2, 5, 64)), dev(bf(1, 2, 5, 64)), dev(i32(1, 4)), dev(i32(1)), dev(i32(1, 1))), "int32 entry"),
    (lambda e: e.kv_append(GOOD, dev(bf(1, 2, 5, 64)), dev(bf(1, 2, 5, 64)), dev(i32(1, 4)), i32(1)), "one device"),
    (lambda e: e.kv_append(GOOD, dev(bf(1, 2, 5, 64)), dev(bf(1, 2, 5, 64)), i32(1, 4), dev(i32(1))), "one device"),
    (lambda e: e.kv_append(GOOD, dev(bf(1, 2, 5, 64)), dev(bf(1, 2, 5, 64)), dev(i32(1, 4)), dev(i32(1)), i32(1)), "one device"),
    (lambda e: e.kv_read(GOOD, dev(i32(1, 4)), dev(i32(2)), 5), "int32 entry"),
    (lambda e: e.kv_read(GOOD, dev(i32(4)), dev(i32(4)), 5), "int32 page table"),
    (lambda e: e.kv_read(GOOD, dev(i32(1, 4)), i32(1), 5), "one device"),
    (lambda e: e.kv_read(GOOD, dev(i32(1, 4)), dev(i32(1)), -1), "max_length"),
    (lambda e: e.kv_read(GOOD, dev(i32(1, 4)), dev(i32(1)), 1 << 30), "max_length"),
    (lambda e: e.paged_attention(dev(bf(1, 3, 64)), GOOD, dev(i32(1, 4)), dev(i32(1))), "BF16 query"),
    (lambda e: e.paged_attention(dev(bf(1, 4, 64)), KVCache(dev(bf(4, 0, 16, 64)), dev(bf(4, 0, 16, 64))), dev(i32(1, 4)), dev(i32(1))), "BF16 query"),
    (lambda e: e.paged_attention(dev(bf(1, 0, 64)), GOOD, dev(i32(1, 4)), dev(i32(1))), "BF16 query"),
    (lambda e: e.paged_attention(dev(bf(1, 4, 32)), GOOD, dev(i32(1, 4)), dev(i32(1))), "BF16 query"),
    (lambda e: e.paged_attention(dev(bf(1, 4, 1, 64)), GOOD, dev(i32(1, 4)), dev(i32(1))), "BF16 query"),
    (lambda e: e.paged_attention(dev(bf(1, 4, 64).half()), GOOD, dev(i32(1, 4)), dev(i32(1))), "BF16 query"),
    (lambda e: e.paged_attention(dev(bf(2, 4, 64)), GOOD, dev(i32(1, 4)), dev(i32(1))), "each sequence"),
    (lambda e: e.paged_attention(dev(bf(1, 4, 64)), GOOD, dev(i32(1, 4)), dev(i32(1)), window=0), "window"),
    (lambda e: e.paged_attention(dev(bf(1, 4, 64)), GOOD, dev(i32(1, 4)), i32(1)), "one device"),
])
def test_wrappers(ext, call, words):
    with pytest.raises(RuntimeError, match=words):
        call(ext)


@pytest.mark.parametrize("scale", [2.0 ** 127, -3e38])
def test_scales_that_overflow(lib, scale):
    """Times log2 e, as scores are scaled, these are infinite, and a score of 0 would be NaN."""
    refused(lib, "uqm_paged_attention", cache(), "2^127", scale=scale)
