"""Refusals of the shared-prefix and page-copy entry points, and their workspace query: on the CPU, before any launch."""
import ctypes

import pytest
import torch

from delta_amd import _lib

A = 1 << 20  # stand-in address, never dereferenced
NO_GPU = pytest.mark.skipif(torch.cuda.is_available(),
                            reason="stand-in addresses: validation-only, run where no GPU is visible")


@pytest.fixture(scope="module", autouse=True)
def lib():
    if not _lib.LIB_PATH.exists():
        from delta_amd import build
        build.build()
    return _lib.load()


def px(row_prefix=A, indptr=A, indices=A, indices_len=16, num=2):
    return ctypes.byref(_lib.SharedPrefixC(row_prefix, indptr, indices, indices_len, num))


def decode(p=px(), q=A, sb=4096, sh=128, kv=A, pages=16, ip=A, ind=A, n=16, last=A, o=A, ob=4096, oh=128, batch=2, hq=32,
           hkv=8, hd=128, dt=0, ws=A, wsb=1 << 40):
    return (p, q, sb, sh, kv, pages, ip, ind, n, last, o, ob, oh, None, batch, hq, hkv, hd, dt, 1.0, 64, ws, wsb, None)


def prefill(qo=A, tokens=5, batch=2, p=px(), ws=A, wsb=1 << 40):
    return (p, A, 4096, 128, A, 16, qo, A, A, 16, A, A, 4096, 128, None, batch, tokens, 5, 32, 8, 128, 0, 1.0, ws, wsb, None)


def copies(caches, n_caches=None, pages=16, hkv=8, hd=128, dt=0, src=A, dst=A, n=3):
    arr = (ctypes.c_void_p * max(len(caches), 1))(*caches)
    return (arr, len(caches) if n_caches is None else n_caches, pages, hkv, hd, dt, src, dst, None, n, None)


def rejects(name, args, match):
    with pytest.raises(_lib.DeltaHipError, match=match):
        _lib.call(name, *args)


def test_empty_calls_return_before_touching_pointers():
    _lib.call("delta_paged_decode_prefix", *decode(p=None, q=None, kv=None, batch=0))
    _lib.call("delta_paged_prefill_prefix", *prefill(qo=None, batch=0))
    _lib.call("delta_paged_prefill_prefix", *prefill(qo=None, tokens=0))
    _lib.call("delta_copy_pages", None, 0, 0, 0, 128, 0, None, None, None, 0, None)
    _lib.call("delta_copy_pages", *copies([None], n=0))


@NO_GPU
@pytest.mark.parametrize("args,match", [
    (dict(hd=64), "head_dim must be 128"),
    (dict(hq=12), "multiple of num_kv_heads"),
    (dict(hq=72), "group size 9 > 8"),
    (dict(dt=7), "bad dtype"),
    (dict(p=None), "null prefix"),
    (dict(batch=1025), "at most 1024 rows and prefixes"),
    (dict(p=px(num=1025)), "at most 1024 rows and prefixes"),
    (dict(p=px(num=-1)), "at most 1024 rows and prefixes"),
    (dict(q=None), "null pointer"),
    (dict(p=px(row_prefix=None)), "null pointer"),
    (dict(p=px(indptr=None)), "null pointer"),
    (dict(p=px(indices=None)), "null pointer"),
    (dict(q=A + 8), "16-byte aligned"),
    (dict(sb=4100), "multiples of 8"),
    (dict(o=A + 2), "o 4-byte aligned"),
    (dict(oh=129), "even strides"),
    (dict(pages=0), "empty cache"),
    (dict(p=px(indices_len=-1)), "bad table lengths"),
    (dict(ws=None), "workspace of .* bytes needed"),
    (dict(wsb=1000), "workspace of .* bytes needed, 1000 given"),
    (dict(ws=A + 16), "workspace must be 256-byte aligned"),
])
def test_decode_prefix(args, match):
    rejects("delta_paged_decode_prefix", decode(**args), match)


@NO_GPU
def test_prefill_prefix():
    rejects("delta_paged_prefill_prefix", prefill(qo=None), "null pointer")
    rejects("delta_paged_prefill_prefix", prefill(p=None), "null prefix")
    rejects("delta_paged_prefill_prefix", prefill(wsb=64), "workspace of .* bytes needed, 64 given")
    rejects("delta_paged_prefill_prefix", prefill(tokens=1 << 40), "too many query tokens")


@NO_GPU
@pytest.mark.parametrize("args,match", [
    (dict(caches=[A], hd=64), "head_dim must be 128"),
    (dict(caches=[A], dt=2), "bad dtype"),
    (dict(caches=[A], hkv=0), "bad num_kv_heads"),
    (dict(caches=[A], pages=0), "bad num_kv_heads or num_pages"),
    (dict(caches=[A], src=None), "null pointer"),
    (dict(caches=[A, None]), "cache 1 null or not 16-byte aligned"),
    (dict(caches=[A, A + 8]), "cache 1 null or not 16-byte aligned"),
    (dict(caches=[A], n=(1 << 23) + 1), "more than 2\\^23 entries"),
])
def test_copy_pages(args, match):
    rejects("delta_copy_pages", copies(**args), match)


def test_workspace_query(lib):
    q = lib.delta_prefix_attention_workspace_bytes
    assert q(0, 32, 8, 100) == 0 and q(4, 12, 8, 100) == 0
    sizes = [q(t, 32, 8, 1025) for t in (1, 8, 32, 128, 1024, 8192)]
    assert all(s > 0 and s % 256 == 0 for s in sizes)
    # a partial per run of a tile, as many as fill the chip; for many tokens two per (token, q head)
    assert max(sizes[:5]) < 100 << 20 and sizes[5] < 8192 * 32 * 2 * 521 * 2
    assert q(32, 32, 8, 4) <= q(32, 32, 8, 1025)
