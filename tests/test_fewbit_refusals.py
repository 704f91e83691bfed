"""CPU: the few-bit entry points check their arguments on the host, before they need a device."""
import ctypes as C
import os
import subprocess

import pytest

INVALID, NOT_INIT = 1, 3
P = 1 << 20          # an address that is never followed: every call here ends on the host


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg.sdq.load_library()


def refused(lib, rc, text):
    assert rc == INVALID, (rc, lib.sdq_last_error())
    assert text in lib.sdq_last_error().decode(), lib.sdq_last_error()


def norm(lib, X=P, dtype=0, ldx=0, res=None, ldr=0, M=4, K=64, w=None, eps=1e-6, sum_=None, lds=0, aq=P, sc=P, h=None, flags=0):
    return lib.sdq_rmsnorm_quantize(X, dtype, ldx, res, ldr, M, K, w, eps, sum_, lds, aq, sc, h, flags, None)


@pytest.mark.parametrize("kw,text", [
    (dict(M=-1), "negative shape"), (dict(K=-5), "negative shape"), (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"),
    (dict(X=None), "null pointer"), (dict(res=P), "go together"), (dict(sum_=P), "go together"),
    (dict(aq=None), "go together"), (dict(sc=None), "go together"), (dict(aq=None, sc=None), "neither"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(ldx=63), "stride"), (dict(res=P, sum_=2 * P, ldr=8), "stride"),
    (dict(res=P, sum_=2 * P, lds=-64), "stride"), (dict(res=2 * P, sum_=P, ldx=96), "in-place"), (dict(flags=0x1), "flag"),
    (dict(X=P + 2), "aligned"), (dict(X=P + 1, dtype=1), "aligned"), (dict(w=P + 2), "aligned"), (dict(sc=P + 1), "aligned"),
])
def test_rmsnorm(lib, kw, text):
    refused(lib, norm(lib, **kw), text)


def test_valid_calls_need_a_device(lib):
    """No CPU path behind the ABI: sound arguments reach the missing device."""
    if lib.sdq_device() >= 0:
        pytest.skip("this process is bound to a GPU")
    assert norm(lib) == NOT_INIT
    h = C.c_uint64()
    assert lib.sdq_w4_upload(P, P, 0, 8, 64, 32, 0, C.byref(h)) == NOT_INIT
    assert lib.sdq_w4_quantize(P, 0, 8, 64, 32, P, P, 0, 0, None) == NOT_INIT
    assert lib.sdq_w4_matmul(1, P, 0, 0, None, 1, P, 0, None, 0, None) == NOT_INIT


@pytest.mark.parametrize("args,text", [
    ((P, 0, 0, 64, 32, P, P, 0, 0), "shape"), ((P, 0, 8, -1, 32, P, P, 0, 0), "shape"), ((P, 0, 8, 64, 48, P, P, 0, 0), "group"),
    ((P, 0, 8, 64, 0, P, P, 0, 0), "group"), ((P, 4, 8, 64, 32, P, P, 0, 0), "src_dtype"), ((P, 3, 8, 64, 32, P, P, 0, 0), "src_dtype"),
    ((P, 0, 8, 64, 32, P, P, 3, 0), "scale_dtype"), ((None, 0, 8, 64, 32, P, P, 0, 0), "null"), ((P, 0, 8, 64, 32, None, P, 0, 0), "null"),
    ((P, 0, 8, 64, 32, P, None, 0, 0), "null"), ((P, 0, 8, 64, 32, P, P, 0, 1), "flag"), ((P + 1, 0, 8, 64, 32, P, P, 0, 0), "aligned"),
    ((P, 0, 1 << 31, 64, 32, P, P, 0, 0), "31 bits"),
])
def test_w4_quantize(lib, args, text):
    refused(lib, lib.sdq_w4_quantize(*args, None), text)


@pytest.mark.parametrize("args,text", [
    ((P, P, 0, 0, 64, 32, 0), "shape"), ((P, P, 0, 8, 0, 32, 0), "shape"), ((P, P, 7, 8, 64, 32, 0), "scale_dtype"),
    ((P, P, 0, 8, 64, 16, 0), "group"), ((None, P, 0, 8, 64, 32, 0), "null"), ((P, None, 0, 8, 64, 32, 0), "null"),
    ((P, P, 0, 8, 64, 32, 0x10), "flag"), ((P, P + 2, 0, 8, 64, 32, 0), "aligned"),
])
def test_w4_upload(lib, args, text):
    h = C.c_uint64()
    refused(lib, lib.sdq_w4_upload(*args, C.byref(h)), text)
    refused(lib, lib.sdq_w4_upload(P, P, 0, 8, 64, 32, 0, None), "null")


@pytest.mark.parametrize("args,text", [
    ((1, P, 0, 0, None, -1, P, 0, None, 0), "negative"), ((1, P, 9, 0, None, 1, P, 0, None, 0), "a_dtype"),
    ((1, P, 0, 0, None, 1, P, 3, None, 0), "out_dtype"), ((1, P, 3, 0, None, 1, P, 0, None, 0), "a_scale"),
    ((1, P, 0, 0, P, 1, P, 0, None, 0), "a_scale"), ((1, None, 0, 0, None, 1, P, 0, None, 0), "null"),
    ((1, P, 0, 0, None, 1, None, 0, None, 0), "null"), ((1, P, 0, 0, None, 1, P, 0, None, 0x2), "flag"),
    ((1, P + 2, 0, 0, None, 1, P, 0, None, 0), "aligned"), ((1, P, 0, 0, None, 1, P, 0, P + 1, 0), "aligned"),
    ((1, P, 0, 0, None, 524281, P, 0, None, 0), "too large"),
])
def test_w4_matmul(lib, args, text):
    refused(lib, lib.sdq_w4_matmul(*args, None), text)


def cache(pkg, **kw):
    d = dict(k=P, v=P, k_scale=P, v_scale=P, pages=4, heads=2, page_size=16, head_dim=64, reserved=0)
    d.update(kw)
    return pkg.sdq.KvCache(**d)


def seqs(pkg, **kw):
    d = dict(row_start=P, kv_len=P, page_table=P, batch=2, max_pages=3)
    d.update(kw)
    return pkg.sdq.KvSeqs(**d)


@pytest.mark.parametrize("ckw,skw,text", [
    (dict(pages=-1), {}, "cache shape"), (dict(heads=0), {}, "cache shape"), (dict(page_size=0), {}, "cache shape"),
    (dict(head_dim=8), {}, "head_dim"), (dict(head_dim=136), {}, "head_dim"), (dict(head_dim=72), {}, "head_dim"),
    (dict(pages=1 << 40), {}, "31 bits"), (dict(pages=1 << 30, heads=1, page_size=2), {}, "31 bits"),
    (dict(k=None), {}, "null pointer in the cache"), (dict(v_scale=None), {}, "null pointer in the cache"),
    (dict(k=P + 8), {}, "16-byte"), (dict(v_scale=P + 2), {}, "aligned"),
    ({}, dict(batch=-1), "sequence table shape"), ({}, dict(batch=1 << 25), "sequence table shape"), ({}, dict(max_pages=-1), "sequence table shape"),
    ({}, dict(max_pages=1 << 30), "sequence table shape"), ({}, dict(row_start=None), "null pointer in the sequence"),
    ({}, dict(kv_len=None), "null pointer in the sequence"), ({}, dict(page_table=None), "null pointer in the sequence"),
    ({}, dict(kv_len=P + 1), "aligned"),
])
def test_kv_descriptors(lib, pkg, ckw, skw, text):
    c, s = cache(pkg, **ckw), seqs(pkg, **skw)
    refused(lib, lib.sdq_kv_append(c, s, P, P, 0, 0, 4, 0, None), text)
    refused(lib, lib.sdq_kv_read(c, s, P, P, 0, 0, 4, 0, None), text)
    refused(lib, lib.sdq_kv_attention(c, s, P, 0, 0, 4, 2, 0.1, P, 0, 0, None), text)


def test_kv_calls(lib, pkg):
    c, s = cache(pkg), seqs(pkg)
    for f in (lib.sdq_kv_append, lib.sdq_kv_read):
        refused(lib, f(None, s, P, P, 0, 0, 4, 0, None), "null descriptor")
        refused(lib, f(c, None, P, P, 0, 0, 4, 0, None), "null descriptor")
        refused(lib, f(c, s, P, P, 3, 0, 4, 0, None), "dtype")
        refused(lib, f(c, s, P, P, 0, 0, -1, 0, None), "rows")
        refused(lib, f(c, s, P, P, 0, 0, 1 << 31, 0, None), "rows")
        refused(lib, f(c, s, None, P, 0, 0, 4, 0, None), "null pointer")
        refused(lib, f(c, s, P, None, 0, 0, 4, 0, None), "null pointer")
        refused(lib, f(c, s, P, P, 0, 127, 4, 0, None), "stride")
        refused(lib, f(c, s, P, P, 0, 0, 4, 0x200, None), "flag")
        refused(lib, f(c, s, P + 2, P, 0, 0, 4, 0, None), "aligned")
    a = lib.sdq_kv_attention
    refused(lib, a(c, s, P, 0, 0, 4, 3, 0.1, P, 0, 0, None), "multiple of the cache's heads")
    refused(lib, a(c, s, P, 0, 0, 4, 0, 0.1, P, 0, 0, None), "multiple of the cache's heads")
    refused(lib, a(c, s, P, 0, 0, 4, 2, 0.0, P, 0, 0, None), "scale")
    refused(lib, a(c, s, P, 0, 0, 4, 2, float("nan"), P, 0, 0, None), "scale")
    refused(lib, a(c, s, P, 0, 0, 4, 2, float("inf"), P, 0, 0, None), "scale")
    refused(lib, a(c, s, P, 0, 0, 1 << 29, 8, 0.1, P, 0, 0, None), "30 bits")
    refused(lib, a(cache(pkg, heads=64), seqs(pkg, batch=1 << 21), P, 0, 0, 4, 64, 0.1, P, 0, 0, None), "26 bits")
    refused(lib, a(c, s, None, 0, 0, 4, 2, 0.1, P, 0, 0, None), "null pointer")
    refused(lib, a(c, s, P, 0, 100, 4, 2, 0.1, P, 0, 0, None), "stride")
    refused(lib, a(c, s, P, 0, 0, 4, 2, 0.1, P, 100, 0, None), "stride")
    refused(lib, a(c, s, P, 0, 0, 4, 2, 0.1, P, 0, 0x4, None), "flag")


def test_places_of_good_and_bad_tables(pkg):
    """The kernels' own index arithmetic, run on the host: nothing leaves the pool."""
    exe = os.path.join(os.path.dirname(pkg.lib_path()), "test_kv_place")
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout
