"""Refusals of the beam-search and paged-cache entry points where sizes end and where there are no rows; helpers as in test_beam_paged_cpu.py."""
import ctypes as C

from test_beam_paged_cpu import ERR, K, P, changed, pool  # noqa: F401


def test_pages_of_no_rows_refuse_bad_counts(K, pkg):
    """Without rows the counts are still read and written."""
    n = K.b200_pages_workspace(0, 10)
    for a, b in ((P + 2049, P + 6144), (P + 2048, P + 6146), (P + 2048, P + 2048), (P + 2048, P + 2048 + 36), (P + 2048 + 36, P + 2048), (None, P + 6144), (P + 2048, None)):
        f, t = (pkg.PageState(refs=r, n_rows=0) for r in (a, b))
        assert K.b200_pages_update(C.byref(pool(pkg)), C.byref(f), C.byref(t), None, None, None, P, P + 8192, n, None) == ERR, (a, b)
        assert K.b200_pages_compact(C.byref(pool(pkg)), C.byref(f), C.byref(t), P + 512, P, P + 8192, n, None) == ERR, (a, b)
