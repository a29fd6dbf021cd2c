"""CPU: argument checks of the C entry points that the attention block adds to
the single calls (no kernel is launched, no pointer read)."""

import ctypes

from preemptlm_b200 import _abi

from .test_attention_cpu import desc, lib  # noqa: F401 (a fixture)


def test_attention_rows(lib):  # noqa: F811
    d = desc()
    n = lib.sg_paged_attention_work_bytes(ctypes.byref(d), 4, 8)
    call = lambda q=16, B=4, t=16, tr=2, w=4, rows=16, ln=16, most=100, out=16, work=16: lib.sg_paged_attention_rows(  # noqa: E731
        ctypes.byref(d), q, 1024, B, 8, t, tr, w, rows, ln, most, 0.1, out, work, n, None)
    for bad in (dict(q=None), dict(t=None), dict(ln=None), dict(out=None), dict(work=None), dict(tr=-1), dict(w=-1), dict(most=-1),
                dict(rows=None)):  # without rows, a table row for every row of q
        assert call(**bad) == _abi.SG_ERR_INVALID_ARG, bad
    assert call(B=0, q=None, t=None, rows=None, tr=0, ln=None, out=None, work=None) == _abi.SG_OK
