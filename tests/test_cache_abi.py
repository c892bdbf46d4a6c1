"""include/hoard_cache.h on the CPU: the library exports what it declares and refuses bad arguments before it touches
CUDA (pointers here are never dereferenced)."""
import ctypes
import os
import re

import pytest

from hoard_b200 import cache, moe

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ONE = ctypes.c_void_p(4096)


def desc(**kw):
    d = dict(n_head=8, n_head_kv=2, head_dim=128, kv_type=1, max_rows=100, max_tokens=4, max_acc_tokens=1, block=16,
             row_stride=0, head_stride=0, scale=0.1)
    d.update(kw)
    return cache.Desc(*[d[f[0]] for f in cache.Desc._fields_])


def query(**kw):
    d = dict(q=4096, qt=1024, qh=128, k=4096, v=4096, vis=0, gate=0, gt=0, gh=0, out=4096, m=1, n_past=10, dev=0)
    d.update(kw)
    return ctypes.create_string_buffer(cache._QUERY.pack(*d.values()), cache._QUERY.size)


def ref(x):
    return ctypes.addressof(x)


def test_header_symbols_exported():
    src = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "hoard_cache.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"^\s*\w+\s+(hoard_kv_\w+)\s*\(", src, flags=re.M)))
    assert names == ["hoard_kv_attention", "hoard_kv_block_attention", "hoard_kv_block_bounds", "hoard_kv_evict",
                     "hoard_kv_store", "hoard_kv_take", "hoard_kv_ws_bytes"]
    assert not [n for n in names if not hasattr(cache._kv(), n)]


@pytest.mark.parametrize("bad", [dict(n_head=0), dict(n_head=9), dict(n_head=130), dict(n_head_kv=0), dict(head_dim=0), dict(head_dim=12),
                                 dict(head_dim=264), dict(kv_type=0), dict(kv_type=12), dict(max_rows=0), dict(max_rows=-1),
                                 dict(max_tokens=0), dict(max_tokens=65), dict(max_tokens=3, max_rows=2),
                                 dict(max_acc_tokens=5), dict(max_acc_tokens=-1), dict(block=8), dict(block=48),
                                 dict(row_stride=100, head_stride=128), dict(row_stride=256, head_stride=64),
                                 dict(row_stride=250, head_stride=128), dict(row_stride=128, head_stride=128),
                                 dict(n_head=4096, n_head_kv=1024, max_tokens=64, max_acc_tokens=0),
                                 dict(scale=3e38), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan"))])
def test_descriptor_refused(bad):
    d = desc(**bad)
    assert cache._kv().hoard_kv_ws_bytes(ref(d)) == -1
    q = query()
    assert cache._kv().hoard_kv_attention(ref(d), ref(q), None, ONE, None) == moe.HOARD_EINVAL


def test_descriptor_accepted():
    L = cache._kv()
    assert L.hoard_kv_ws_bytes(None) == -1
    for ok in (dict(), dict(row_stride=512, head_stride=128), dict(row_stride=128, head_stride=12800), dict(block=0), dict(head_dim=8),
               dict(max_tokens=64, max_acc_tokens=0), dict(n_head=4096, n_head_kv=1024, max_tokens=63, max_acc_tokens=0)):
        assert L.hoard_kv_ws_bytes(ref(desc(**ok))) > 0
    # a workspace for more tokens is not smaller
    sizes = [L.hoard_kv_ws_bytes(ref(desc(max_tokens=t, max_acc_tokens=0))) for t in (1, 4, 16, 64)]
    assert sizes == sorted(sizes)


@pytest.mark.parametrize("bad", [dict(q=0), dict(k=0), dict(v=0), dict(out=0), dict(k=4104), dict(v=4100), dict(m=0), dict(m=5),
                                 dict(n_past=-1), dict(n_past=100), dict(m=2, n_past=99), dict(qh=64), dict(qt=-1),
                                 dict(m=2, qt=512), dict(m=2, qt=128, qh=255), dict(m=2, qt=64, qh=4096), dict(gate=4096, gh=64), dict(gate=4096, gh=128, gt=-1)])
def test_query_refused(bad):
    d, q = desc(), query(**bad)
    L = cache._kv()
    assert L.hoard_kv_attention(ref(d), ref(q), None, ONE, None) == moe.HOARD_EINVAL
    assert L.hoard_kv_block_attention(ref(d), ref(q), ONE, 1, 1, 1, None, ONE, None) == moe.HOARD_EINVAL


def test_other_refusals():
    L, d, q, E = cache._kv(), desc(), query(), moe.HOARD_EINVAL
    assert L.hoard_kv_attention(ref(d), ref(q), None, None, None) == E                      # no workspace
    assert L.hoard_kv_attention(ref(d), ref(q), None, ctypes.c_void_p(4097), None) == E     # misaligned
    assert L.hoard_kv_attention(ref(d), None, None, ONE, None) == E
    q2 = query(m=2)
    assert L.hoard_kv_attention(ref(d), ref(q2), ONE, ONE, None) == E                       # m > max_acc_tokens
    none = desc(block=0)
    assert L.hoard_kv_block_attention(ref(none), ref(q), ONE, 1, 1, 1, None, ONE, None) == E
    assert L.hoard_kv_block_bounds(ref(none), ONE, ONE, 0, 16, None, None) == E
    for n_sink, n_local, n_sel in ((-1, 1, 1), (0, 0, 1), (0, 1, -1)):
        assert L.hoard_kv_block_attention(ref(d), ref(q), ONE, n_sink, n_local, n_sel, None, ONE, None) == E
    for row0, row1 in ((-1, 5), (6, 5), (0, 101)):
        assert L.hoard_kv_block_bounds(ref(d), ONE, ONE, row0, row1, None, None) == E
    ev = lambda rows, keep, **k: L.hoard_kv_evict(ref(d), k.get("kc", ONE), ONE, ONE, ONE, rows, keep, 0, 50, ONE, ONE, ONE, None)
    assert ev(101, 5) == E and ev(10, 0) == E and ev(10, 11) == E and ev(10, 5, kc=None) == E and ev(10, 5, kc=ctypes.c_void_p(8)) == E
    path = lambda *p: (ctypes.c_int32 * len(p))(*p)
    take = lambda row0, p, n: L.hoard_kv_take(ref(d), ONE, ONE, row0, p, n, None)
    assert take(0, path(1, 1), 2) == E and take(0, path(2, 1), 2) == E and take(0, path(-1, 1), 2) == E
    assert take(0, path(0, 64), 2) == E and take(95, path(0, 5), 2) == E and take(-1, path(0, 1), 2) == E and take(0, None, 1) == E
    assert take(5, None, 0) == 0 and take(5, path(0, 1, 2), 3) == 0                         # nothing to move, nothing launched
    st = lambda **k: L.hoard_kv_store(ref(d), ONE, 1024, k.get("qh", 128), ONE, ONE, k.get("qn", ONE), ONE, k.get("mode", 2), 1e-6,
                                      k.get("rope", 128), k.get("base", 1e4), ONE, k.get("m", 1), k.get("row0", 0), None,
                                      k.get("out", ctypes.c_void_p(8192)), ONE, ONE, None, None, None)
    for bad in (dict(mode=3), dict(mode=2, qn=None), dict(rope=0), dict(rope=127), dict(rope=130), dict(base=0.0), dict(m=0), dict(m=65),
                dict(row0=-1), dict(out=ONE), dict(qh=64), dict(mode=1, qh=256)):
        assert st(**bad) == E, bad


def test_tree_visibility():
    words, depth = cache.tree_visibility([-1, 0, 0, 1, -1, 4])
    assert words == [1, 3, 5, 11, 16, 48] and depth == [0, 1, 1, 2, 0, 1]
    words, depth = cache.tree_visibility(list(range(-1, 63)))
    assert words[62] == 2**63 - 1 and words[63] == -1 and depth[63] == 63
    for bad in ([], [0], [-2], [-1, 1], [-1] * 65):
        with pytest.raises(ValueError):
            cache.tree_visibility(bad)
