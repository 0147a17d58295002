"""What the paged cache's operators and C entry points refuse, and the arithmetic of slots and pages by which the kernels stay inside the pool, without a GPU."""
import ctypes
import os
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Strided(ctypes.Structure):
    _fields_ = [("ptr", ctypes.c_void_p), ("batch", ctypes.c_int64), ("head", ctypes.c_int64), ("row", ctypes.c_int64)]


class Cache(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("k", "v", "positions", "weights", "table", "lengths")] + [("pages", ctypes.c_int64)] + [
        (n, ctypes.c_int32) for n in ("kv_heads", "page_size", "batch", "max_pages")]


A = 0x1000
GOOD = dict(k=A, v=A, positions=A, weights=A, table=A, lengths=A, pages=10, kv_heads=2, page_size=16, batch=3, max_pages=4)


def _cache(**change):
    return ctypes.byref(Cache(**dict(GOOD, **change)))


def _lib():
    from flex_block_attn_amd import _lib

    return _lib.load()


ROW = Strided(A, 256, 128, 128)


@pytest.mark.parametrize("change,code,text", [
    (dict(k=None), 1, "cache k"), (dict(v=0x1008), 1, "aligned"), (dict(pages=0), 1, "positive"), (dict(max_pages=0), 1, "positive"), (dict(batch=0), 1, "positive"),
    (dict(page_size=8), 1, "page_size"), (dict(page_size=48), 1, "page_size"), (dict(table=None), 1, "table"), (dict(lengths=None), 1, "lengths"), (dict(weights=0x1004), 1, "weights"), (dict(positions=0x1008), 1, "positions"),
    (dict(max_pages=1 << 25), 2, "2^28"), (dict(pages=1 << 31), 2, "slots"), (dict(page_size=256, max_pages=1 << 20, batch=256), 2, "2^35"),
])
def test_c_entries_refuse_a_cache(change, code, text):
    lib = _lib()
    c = _cache(**change)
    q, f = ctypes.byref(ROW), ctypes.c_void_p(A)
    for call in (lambda: lib.fba_cache_attn(c, q, q, 4, 1 << 30, 0, 0, 0, f, 1 << 40, None), lambda: lib.fba_cache_append(c, q, q, None, None, None, 1, ctypes.c_void_p(0x2000), None),
                 lambda: lib.fba_cache_evict(c, 8, 0, 0, ctypes.c_void_p(0x2000), f, 1 << 40, None)):
        assert call() == code
        assert text in lib.fba_last_error().decode()


def test_c_entries_refuse_arguments():
    lib = _lib()
    c, q, f, out = _cache(), ctypes.byref(ROW), ctypes.c_void_p(A), ctypes.c_void_p(0x2000)
    much = 1 << 40
    for code, text, call in [
        (1, "heads", lambda: lib.fba_cache_attn(c, q, q, 3, 99, 0, 0, 0, f, much, None)),
        (1, "type", lambda: lib.fba_cache_attn(c, q, q, 4, 99, 0, 0, 2, f, much, None)),
        (1, "window", lambda: lib.fba_cache_attn(c, q, q, 4, 0, 0, 0, 0, f, much, None)),
        (1, "sinks", lambda: lib.fba_cache_attn(c, q, q, 4, 99, -1, 0, 0, f, much, None)),
        (1, "whole cache", lambda: lib.fba_cache_attn(c, q, q, 4, 10, 0, 1, 0, f, much, None)),
        (1, "ws must", lambda: lib.fba_cache_attn(c, q, q, 4, 99, 0, 0, 0, f, 64, None)),
        (1, "weights is null", lambda: lib.fba_cache_attn(_cache(weights=None), q, q, 4, 99, 0, 1, 0, f, much, None)),
        (1, "q is null", lambda: lib.fba_cache_attn(c, None, q, 4, 99, 0, 0, 0, f, much, None)),
        (1, "tokens", lambda: lib.fba_cache_append(c, q, q, None, None, None, 0, out, None)),
        (1, "lengths_out", lambda: lib.fba_cache_append(c, q, q, None, None, None, 1, None, None)),
        (1, "lengths_out must not", lambda: lib.fba_cache_append(c, q, q, None, None, None, 1, f, None)),
        (1, "k: strides", lambda: lib.fba_cache_append(c, ctypes.byref(Strided(A, 4, 0, 128)), q, None, None, None, 1, out, None)),
        (1, "budget", lambda: lib.fba_cache_evict(c, 0, 0, 0, out, f, much, None)),
        (1, "fit the budget", lambda: lib.fba_cache_evict(c, 8, 5, 4, out, f, much, None)),
        (1, "fit the budget", lambda: lib.fba_cache_evict(c, 8, -1, 4, out, f, much, None)),
        (1, "positions or weights", lambda: lib.fba_cache_evict(_cache(positions=None), 8, 0, 0, out, f, much, None)),
        (1, "ws must", lambda: lib.fba_cache_evict(c, 8, 0, 0, out, f, 4, None)),
        (1, "ws must", lambda: lib.fba_cache_evict(c, 8, 0, 0, out, None, much, None)),
    ]:
        assert call() == code, text
        assert text in lib.fba_last_error().decode()
    assert lib.fba_cache_attn_workspace_bytes(c, 3, 0) == -1
    assert lib.fba_cache_evict_workspace_bytes(c, 0) == -1
    # scores of every head and slot, where weights are added up
    assert lib.fba_cache_attn_workspace_bytes(c, 4, 1) - lib.fba_cache_attn_workspace_bytes(c, 4, 0) == 3 * 4 * 64 * 4


def test_python_refuses_without_a_gpu():
    import flex_block_attn_amd as fba

    z = lambda *shape, dtype=torch.bfloat16: torch.zeros(shape, dtype=dtype)
    cache = fba.PagedCache(z(4, 2, 16, 128), z(4, 2, 16, 128))
    table, n = z(1, 2, dtype=torch.int32), z(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU tensor"):
        fba.cache_attn_func(z(1, 2, 1, 128), cache, table, n)
    with pytest.raises(ValueError, match="GPU tensor"):
        fba.cache_append(cache, table, n, z(1, 2, 1, 128), z(1, 2, 1, 128))
    with pytest.raises(ValueError, match="GPU tensor"):
        fba.cache_evict(cache, table, n, 4)
    with pytest.raises(TypeError, match="PagedCache"):
        fba.cache_evict((cache.k, cache.v), table, n, 4)
    for size in (0, 8, 24):
        with pytest.raises(ValueError, match="page_size"):
            fba.paged_cache(4, 2, size, device="cpu")
    with pytest.raises(TypeError, match="dtype"):
        fba.paged_cache(4, 2, 16, dtype=torch.float32, device="cpu")
    with pytest.raises(ValueError, match="pages"):
        fba.paged_cache(0, 2, 16, device="cpu")


PROBE = """
#include "fba_cache.h"
extern "C" {
int holds(int page_log2, int max_pages, long long n) { fba::CacheView c{}; c.page_log2 = page_log2; c.max_pages = max_pages; return c.holds(n); }
int page_of(const int* table, long long pages, int page_log2, int max_pages, int b, int slot) {
  fba::CacheView c{}; c.table = table; c.pages = pages; c.page_log2 = page_log2; c.max_pages = max_pages; return c.page_of(b, slot);
}
long long row_of(int kv_heads, int page_log2, int page, int head, int slot) { fba::CacheView c{}; c.kv_heads = kv_heads; c.page_log2 = page_log2; return c.row_of(page, head, slot); }
}
"""


@pytest.fixture(scope="module")
def probe(tmp_path_factory):
    """The kernels' own slot arithmetic, compiled for the host."""
    at = tmp_path_factory.mktemp("pages")
    (at / "probe.cpp").write_text(PROBE)
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__=1", f"-I{rocm}/include", "-I" + os.path.join(ROOT, "flex_block_attn_amd", "csrc"),
                    str(at / "probe.cpp"), "-o", str(at / "probe.so")], check=True, capture_output=True)
    lib = ctypes.CDLL(str(at / "probe.so"))
    lib.row_of.restype = ctypes.c_longlong
    lib.holds.argtypes = [ctypes.c_int, ctypes.c_int, ctypes.c_longlong]
    lib.page_of.argtypes = [ctypes.c_void_p, ctypes.c_longlong] + [ctypes.c_int] * 4
    return lib


def test_slots_and_pages(probe):
    assert [probe.holds(4, 3, n) for n in (-1, 0, 1, 48, 49, 1 << 40)] == [0, 1, 1, 1, 0, 0]
    assert probe.holds(14, 1 << 14, 1 << 28) == 1 and probe.holds(14, 1 << 14, (1 << 28) + 1) == 0  # in 64 bits
    table = (ctypes.c_int * 6)(0, 9, 10, -1, 7, 1 << 30)
    of = lambda b, slot: probe.page_of(table, 10, 4, 3, b, slot)
    assert [of(0, 0), of(0, 15), of(0, 16), of(0, 32), of(1, 0), of(1, 16), of(1, 47)] == [0, 0, 9, -1, -1, 7, -1]
    assert probe.row_of(3, 4, 0, 0, 0) == 0 and probe.row_of(3, 4, 2, 1, 37) == (2 * 3 + 1) * 16 + 5
    assert probe.row_of(65535, 14, 0x7ffffffe, 65534, 16383) == (0x7ffffffe * 65535 + 65534) * 16384 + 16383  # in 64 bits


@pytest.mark.gpu
def test_python_refuses_on_the_gpu(gpu):
    import flex_block_attn_amd as fba
    from flex_block_attn_amd import _lib

    z = lambda *shape, dtype=torch.bfloat16: torch.zeros(shape, dtype=dtype, device=gpu)
    i32 = torch.int32
    cache = fba.paged_cache(4, 2, 16, device=gpu, evicting=True)
    plain = fba.PagedCache(cache.k, cache.v)
    table, n, q, k = z(3, 2, dtype=i32), z(3, dtype=i32), z(3, 4, 1, 128), z(3, 2, 5, 128)
    attend, append, evict = fba.cache_attn_func, fba.cache_append, fba.cache_evict
    for error, text, call in [
        (TypeError, "bfloat16 or float16", lambda: attend(q, fba.PagedCache(cache.k.float(), cache.v.float()), table, n)),
        (TypeError, "bfloat16 or float16", lambda: attend(q, fba.PagedCache(cache.k, cache.v.half()), table, n)),
        (ValueError, "shape", lambda: attend(q, fba.PagedCache(cache.k, cache.v[:3]), table, n)),
        (ValueError, "contiguous", lambda: attend(q, fba.PagedCache(cache.k.transpose(0, 1), cache.v.transpose(0, 1)), table, n)),
        (ValueError, "page_size", lambda: attend(q, fba.PagedCache(z(4, 2, 24, 128), z(4, 2, 24, 128)), table, n)),
        (ValueError, "page and a head", lambda: attend(q, fba.PagedCache(z(0, 2, 16, 128), z(0, 2, 16, 128)), table, n)),
        (ValueError, "weights", lambda: attend(q, fba.PagedCache(cache.k, cache.v, weights=z(4, 2, 8, dtype=torch.float32)), table, n)),
        (ValueError, "positions", lambda: evict(fba.PagedCache(cache.k, cache.v, cache.positions.long(), cache.weights), table, n, 4)),
        (ValueError, "table", lambda: attend(q, cache, table.long(), n)),
        (ValueError, "table", lambda: attend(q, cache, table[0], n)),
        (ValueError, "lengths", lambda: attend(q, cache, table, n[:2])),
        (ValueError, "lengths", lambda: attend(q, cache, table, n.long())),
        (ValueError, "GPU tensor", lambda: attend(q, cache, table.cpu(), n)),
        (TypeError, "tensor", lambda: attend(q, cache, [[0, 1]], n)),
        (_lib.FbaError, "2\\^28", lambda: attend(z(1, 4, 1, 128), cache, z(1, (1 << 24) + 1, dtype=i32), n[:1])),
        (TypeError, "q must have the cache's", lambda: attend(q.half(), cache, table, n)),
        (ValueError, "q must have shape", lambda: attend(z(3, 4, 2, 128), cache, table, n)),
        (ValueError, "q must have shape", lambda: attend(z(2, 4, 1, 128), cache, table, n)),
        (ValueError, "multiple", lambda: attend(z(3, 3, 1, 128), cache, table, n)),
        (ValueError, "with weights", lambda: attend(q, plain, table, n, accumulate=True)),
        (ValueError, "window must be None", lambda: attend(q, cache, table, n, window=8, accumulate=True)),
        (ValueError, "window", lambda: attend(q, cache, table, n, window=0)),
        (TypeError, "window", lambda: attend(q, cache, table, n, window=2.0)),
        (ValueError, "sinks", lambda: attend(q, cache, table, n, sinks=-1)),
        (ValueError, "no_grad", lambda: attend(q.clone().requires_grad_(True), cache, table, n)),
        (TypeError, "k must have", lambda: append(cache, table, n, k.half(), k.half())),
        (ValueError, "k and v must have shape", lambda: append(cache, table, n, k[:2], k[:2])),
        (ValueError, "k and v must have shape", lambda: append(cache, table, n, k, k[:, :, :4])),
        (ValueError, "counts", lambda: append(cache, table, n, k, k, counts=n.long())),
        (ValueError, "positions", lambda: append(cache, table, n, k, k, positions=n[:1])),
        (ValueError, "has none", lambda: append(plain, table, n, k, k, positions=n)),
        (ValueError, "has none", lambda: append(plain, table, n, k, k, weights=z(3, 2, 5, dtype=torch.float32))),
        (ValueError, "weights must", lambda: append(cache, table, n, k, k, weights=z(3, 2, 4, dtype=torch.float32))),
        (ValueError, "no_grad", lambda: append(cache, table, n, k.clone().requires_grad_(True), k)),
        (ValueError, "positions and weights", lambda: evict(plain, table, n, 4)),
        (ValueError, "budget", lambda: evict(cache, table, n, 0)),
        (TypeError, "budget", lambda: evict(cache, table, n, None)),
        (ValueError, "fit the budget", lambda: evict(cache, table, n, 4, recent=3, sinks=2)),
        (ValueError, "recent", lambda: evict(cache, table, n, 4, recent=-1)),
    ]:
        with pytest.raises(error, match=text):
            call()
    assert append(cache, table, n, k[:, :, :0], k[:, :, :0]).tolist() == [0, 0, 0]
    with torch.no_grad():
        assert int(attend(q.clone().requires_grad_(True), cache, table, n).count_nonzero()) == 0
