"""The C-ABI library loads and exports every entry point include/sokutou_b200.h declares; argument
validation answers with error codes before touching any device (no GPU needed)."""

import ctypes
import os
import re

import pytest

from conftest import ROOT

HEADER = os.path.join(ROOT, "include", "sokutou_b200.h")


def declared_symbols():
    src = open(HEADER).read()
    return sorted(set(re.findall(r"^SK_API\s+(?:int|size_t)\s+(sk_\w+)\s*\(", src, re.M)))


def test_header_declares_the_boundary():
    syms = declared_symbols()
    for s in ("sk_dit_attention", "sk_dit_qkv_prologue", "sk_decode_attention", "sk_decode_workspace_bytes",
              "sk_device_error", "sk_version"):
        assert s in syms


def test_library_exports_every_declared_symbol(native_lib):
    for s in declared_symbols():
        assert hasattr(native_lib, s), s
    from sokutou_b200 import _lib
    assert set(_lib.SIGNATURES) == set(declared_symbols())


def test_version(native_lib):
    assert native_lib.sk_version() >= 100


def test_argument_errors_without_device(native_lib):
    P = ctypes.c_void_p
    fake = P(4096)  # never dereferenced: validation fails first
    # null q
    assert native_lib.sk_dit_attention(None, fake, fake, None, None, None, fake, 1, 1, 1, 1, 0, 64, 0, 0, 0, 0.0, None) == -1
    # unsupported head dim
    assert native_lib.sk_dit_attention(fake, fake, fake, None, None, None, fake, 1, 1, 1, 1, 0, 96, 0, 0, 0, 0.0, None) == -2
    # misaligned pointer
    assert native_lib.sk_dit_attention(P(4100), fake, fake, None, None, None, fake, 1, 1, 1, 1, 0, 64, 0, 0, 0, 0.0, None) == -1
    # unsupported dtype
    assert native_lib.sk_dit_attention(fake, fake, fake, None, None, None, fake, 1, 1, 1, 1, 0, 64, 0, 0, 7, 0.0, None) == -2
    # decode: nq must be 2*nkv, hd 128
    f = ctypes.c_float
    assert native_lib.sk_decode_attention(fake, fake, fake, f(1e-6), fake, fake, fake, None, 0, 16, 4, 4, 128, fake,
                                          None, 0, 0, None) == -2
    assert native_lib.sk_decode_attention(fake, fake, fake, f(1e-6), fake, fake, fake, None, 0, 16, 4, 2, 64, fake,
                                          None, 0, 0, None) == -2
    # decode: split-KV needs a workspace when max_len spans several chunks
    assert native_lib.sk_decode_attention(fake, fake, fake, f(1e-6), fake, fake, fake, None, 0, 1024, 4, 2, 128, fake,
                                          None, 0, 0, None) == -5
    assert native_lib.sk_decode_workspace_bytes(1024, 16, 8, 128, 0) > 0
    assert native_lib.sk_decode_workspace_bytes(0, 16, 8, 128, 0) == 0


def test_ops_raise_on_missing_library(monkeypatch, tmp_path):
    from sokutou_b200 import _lib
    monkeypatch.setattr(_lib, "_lib", None)
    monkeypatch.setattr(_lib, "LIB_PATH", str(tmp_path / "missing.so"))
    with pytest.raises(_lib.SokutouError):
        _lib.lib()


def _shared(**kw):
    """A well-formed SkSharedDecode over addresses that are never dereferenced."""
    from sokutou_b200 import _lib
    d = dict(Kp=1 << 20, Vp=2 << 20, prefix_head_stride=100 * 128, prefix_row_stride=128, Kc=3 << 20, Vc=4 << 20,
             request_stride=8 * 64 * 128, head_stride=64 * 128, row_stride=128, mass=None, rope=5 << 20, pos=6 << 20,
             rows=7 << 20, workspace=8 << 20, ws_bytes=1 << 40, qkv_stride=32 * 128, out_stride=16 * 128, R=4, nq=16,
             nkv=8, hd=128, prefix_len=100, max_len=64, rope_len=200, cache_dtype=0, qkv_dtype=1, out_dtype=1, eps=1e-6)
    return _lib.SkSharedDecode(**(d | kw))


def test_shared_decode_refusals_without_device(native_lib):
    def call(qkv=1 << 22, qn=1 << 23, kn=1 << 23, out=1 << 24, **kw):
        return native_lib.sk_decode_attention_shared(ctypes.byref(_shared(**kw)), qkv, qn, kn, out, None)

    size = lambda **kw: native_lib.sk_decode_shared_workspace_bytes(ctypes.byref(_shared(**kw)))  # noqa: E731
    assert native_lib.sk_decode_attention_shared(None, 16, 16, 16, 16, None) == -1
    assert native_lib.sk_decode_shared_workspace_bytes(None) == 0
    for kw in (dict(R=0), dict(nkv=0), dict(nq=0), dict(prefix_len=-1), dict(max_len=0), dict(rope_len=0)):
        assert call(**kw) == -1 and size(**kw) == 0, kw
    for kw in (dict(hd=96), dict(nq=17), dict(nq=72), dict(R=1025), dict(cache_dtype=2), dict(nkv=2000, nq=2000)):
        assert call(**kw) == -2 and size(**kw) == 0, kw
    for kw in (dict(qkv_dtype=7), dict(out_dtype=2), dict(cache_dtype=1, out_dtype=0), dict(cache_dtype=1, qkv_dtype=0)):
        assert call(**kw) == -2, kw
    for kw in (dict(qkv=None), dict(qn=None), dict(kn=None), dict(out=None), dict(rope=None), dict(pos=None), dict(Kc=None),
               dict(Vc=None), dict(Kp=None), dict(Vp=None), dict(qkv=(1 << 22) + 4), dict(Kc=(3 << 20) + 8), dict(pos=(6 << 20) + 4),
               dict(row_stride=127), dict(row_stride=132), dict(head_stride=8), dict(request_stride=0),
               dict(prefix_row_stride=64), dict(prefix_head_stride=130), dict(qkv_stride=31 * 128), dict(out_stride=16 * 128 + 1),
               dict(mass=8, mass_request_stride=0, mass_head_stride=64), dict(mass=6)):
        assert call(**kw) == -1, kw
    assert call(workspace=None) == -5 and call(workspace=(8 << 20) + 16) == -5 and call(ws_bytes=size() - 1) == -5
    # out over qkv, one row of it, one element of it; then side by side in rows of 48 * 128, which only a device is missing for
    at, wide = 1 << 22, dict(qkv_stride=48 * 128, out_stride=48 * 128)
    for kw in (dict(out=at), dict(out=at + 3 * 32 * 128 * 4), dict(out=at - 4 * 16 * 128 * 4 + 16), dict(out=at, R=1),
               dict(out=at + 32 * 128 * 4 - 16, **wide), dict(out=at - 16 * 128 * 4 + 16, **wide)):
        assert call(qkv=at, **kw) == -1, kw
    for kw in (dict(out=at + 32 * 128 * 4, **wide), dict(out=at - 16 * 128 * 4, **wide), dict(out=at + 4 * 32 * 128 * 4)):
        assert call(qkv=at, ws_bytes=0, **kw) == -5, kw
    assert size() > 0 and size(mass=256) > size() > size(prefix_len=0) and size(R=5) > size()


def test_cache_evict_refusals_without_device(native_lib):
    from sokutou_b200 import _lib
    kv, ms = ctypes.c_longlong * 4, ctypes.c_longlong * 3

    def desc(**kw):
        d = dict(K=1 << 30, V=2 << 30, mass=3 << 30, kv_stride=kv(4 * 2 * 100 * 64, 2 * 100 * 64, 100 * 64, 64),
                 mass_stride=ms(800, 200, 100), K_out=4 << 30, V_out=5 << 30, mass_out=6 << 30,
                 kv_out_stride=kv(4 * 2 * 100 * 64, 2 * 100 * 64, 100 * 64, 64), mass_out_stride=ms(800, 200, 100),
                 rows=7 << 30, rows_out=7 << 30, workspace=8 << 30, ws_bytes=1 << 40, N=3, R=4, nkv=2, hd=64, max_len=100,
                 max_len_out=100, keep=50, first=10, recent=20, cache_dtype=0)
        return ctypes.byref(_lib.SkCacheEvict(**(d | kw)))

    call = lambda **kw: native_lib.sk_cache_evict(desc(**kw), None)  # noqa: E731
    size = lambda **kw: native_lib.sk_cache_evict_workspace_bytes(desc(**kw))  # noqa: E731
    assert native_lib.sk_cache_evict(None, None) == -1 and native_lib.sk_cache_evict_workspace_bytes(None) == 0
    for kw in (dict(N=0), dict(R=0), dict(nkv=0), dict(max_len=0), dict(keep=0), dict(keep=101), dict(max_len_out=49),
               dict(first=-1), dict(recent=-1), dict(first=31)):
        assert call(**kw) == -1 and size(**kw) == 0, kw
    for kw in (dict(hd=80), dict(cache_dtype=2), dict(max_len=1 << 22), dict(N=1 << 20, R=1 << 10, nkv=4)):
        assert call(**kw) == -2 and size(**kw) == 0, kw
    for name in ("K", "V", "mass", "K_out", "V_out", "mass_out", "rows", "rows_out"):
        assert call(**{name: None}) == -1, name
        assert call(**{name: (9 << 30) + 2}) == -1, name
    for kw in (dict(kv_stride=kv(51200, 12800, 6400, 32)), dict(kv_out_stride=kv(51200, 12800, 6404, 64)),
               dict(mass_stride=ms(800, 0, 100)), dict(K_out=1 << 30), dict(mass_out=3 << 30),
               # in place at other strides; a destination that meets the source
               dict(K_out=1 << 30, V_out=2 << 30, mass_out=3 << 30, mass_out_stride=ms(801, 200, 100)),
               dict(K_out=(1 << 30) + 128), dict(V_out=(1 << 30) - 64 * 2), dict(mass_out=(3 << 30) + 400),
               dict(mass_out=(1 << 30) + 400)):
        assert call(**kw) == -1, kw
    assert call(workspace=None) == -5 and call(ws_bytes=size() - 1) == -5
    assert size() >= 3 * 4 * 2 * 50 * 4
