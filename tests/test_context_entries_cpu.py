"""C entries of window attention and the paged cache with arguments that they refuse or that leave nothing to do: host code,
checked without a GPU, in a process of its own."""
import subprocess
import sys
import textwrap

import pytest

from tinyinfinitrain_b200._build import KERNEL_LIB

PRELUDE = f"""
import ctypes as c
lib = c.CDLL({str(KERNEL_LIB)!r})
P, I, L, F = c.c_void_p, c.c_int, c.c_longlong, c.c_float
class Attn(c.Structure):
    _fields_ = [(n, P) for n in "q k v o lse d_o dq dk dv delta dq_accum".split()] + [(n, I) for n in "B T Hq Hkv hd".split()] + \\
        [(n + "_stride_t", L) for n in "q k v o dq dk dv do".split()] + [("scale", F)]
class Window(c.Structure):
    _fields_ = [("attn", Attn), ("window", I), ("sinks", I), ("dtype", I), ("workspace", P), ("o_lo", P)]
class Cache(c.Structure):
    _fields_ = [("k_cache", P), ("v_cache", P), ("page_table", P), ("table_stride", L)] + \\
        [(n, I) for n in "table_width n_pages page_size B Hq Hkv hd window sinks dtype".split()]
for f in (lib.titb_window_attn_bwd_workspace, lib.titb_paged_attention_workspace):
    f.restype = L
def window(**kw):
    w = Window(window=4, sinks=1, dtype=1)
    for n, v in dict(B=2, T=300, Hq=4, Hkv=2, hd=64, scale=1.0, **{{n + "_stride_t": 512 for n in "q k v o dq dk dv do".split()}}).items():
        setattr(w.attn, n, v)
    for n, v in kw.items():
        setattr(w if n in ("window", "sinks", "dtype", "o_lo") else w.attn, n, v)
    return w
def cache(**kw):
    d = Cache(table_stride=8, table_width=8, n_pages=100, page_size=16, B=2, Hq=8, Hkv=2, hd=64, window=2 ** 31 - 1, sinks=0, dtype=1)
    for n, v in kw.items():
        setattr(d, n, v)
    return d
def append(d, qkv=None, T=1, stride=1024):
    return lib.titb_cache_append(c.byref(d), P(qkv), L(stride), L(stride), T, P(None), P(None), c.c_double(1e4), P(None), P(None), P(None))
def paged(d, q=None, stride=512):
    return lib.titb_paged_attention(c.byref(d), P(q), L(stride), P(None), F(1.0), P(None), P(None), P(None))
SHAPE, ALIGN = 20003, 20001
"""


def _run(body):
    code = PRELUDE + textwrap.dedent(body)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("entry", ["titb_window_attn_fwd", "titb_window_attn_bwd"])
def test_window_attention(entry):
    _run(f"""
    f = lambda **kw: lib.{entry}(c.byref(window(**kw)), P(None))
    for kw in (dict(B=0), dict(T=0), dict(Hq=0)):
        assert f(**kw) == 0, kw
    for kw in (dict(hd=0), dict(hd=136), dict(hd=12), dict(Hkv=0), dict(Hkv=3), dict(window=0), dict(window=-5), dict(sinks=-1),
               dict(T=2 ** 21), dict(Hq=2 ** 30, Hkv=2)):
        assert f(**kw) == SHAPE, kw
    for kw in (dict(q=8), dict(k=2), dict(v=4), dict(o=8), dict(o_lo=4), dict(q_stride_t=516), dict(o_stride_t=4)):
        assert f(**kw) == ALIGN, kw
    assert lib.titb_window_attn_bwd_workspace(c.byref(window(Hkv=0))) == 0
    """)


def test_window_attention_workspace():
    """The dQ accumulator, and parts of the sinks' blocks only where there are several."""
    _run("""
    size = lambda **kw: lib.titb_window_attn_bwd_workspace(c.byref(window(**kw)))
    assert size(sinks=0) == 2 * 300 * 4 * 64 and size(sinks=0, dtype=0) == 0
    assert size(T=20000) > 2 * 20000 * 4 * 64 and size(T=20000, dtype=0) > 0
    assert size(T=20000, window=20000) == 2 * 20000 * 4 * 64
    assert size(window=2 ** 31 - 1, sinks=2 ** 31 - 1) == 2 * 300 * 4 * 64
    """)


def test_cache():
    _run("""
    for f in (append, paged):
        assert f(cache(B=0)) == 0
        for kw in (dict(hd=0), dict(hd=136), dict(hd=4), dict(Hkv=0), dict(Hkv=3), dict(page_size=0), dict(table_width=-1), dict(n_pages=-1),
                   dict(n_pages=2 ** 30), dict(window=0), dict(sinks=-1), dict(dtype=2)):
            assert f(cache(**kw)) == SHAPE, (f, kw)
        assert f(cache(k_cache=8)) == ALIGN and f(cache(v_cache=8)) == ALIGN
        assert f(cache(), 8) == ALIGN and f(cache(), stride=1028) == ALIGN
    assert append(cache(), T=0) == 0
    assert append(cache(B=2 ** 16), T=2 ** 16) == SHAPE
    assert paged(cache(Hq=0)) == 0
    """)


def test_cache_workspace():
    """None where no sequence can take more than a tile; bounded by the card, not by the cache."""
    _run("""
    size = lambda **kw: lib.titb_paged_attention_workspace(c.byref(cache(**kw)))
    assert size(table_width=4) == 0 and size(window=60, sinks=4, table_width=1000) == 0 and size(table_width=0) == 0
    assert size(Hkv=0) == 0
    big = size(table_width=2 ** 20, B=1000, n_pages=2 ** 20)
    assert size() == 0 and 0 < size(table_width=9) <= big < 32 << 20 and size(table_width=2 ** 24, B=4000, n_pages=2 ** 20) == big
    """)
