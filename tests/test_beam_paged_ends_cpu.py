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


def test_pages_refuse_more_pages_than_they_can_number(K, pkg):
    """Beyond 2^30 pages, 32-bit positions in the lists of pages would overflow."""
    most = 1 << 30
    assert K.b200_pages_workspace(1, most) > 0 and K.b200_pages_workspace(1, most + 1) == 0
    for n_pages in (most + 1, (1 << 31) - 1):
        f, t = (pkg.PageState(tables=P + i, lens=P + i + 256, refs=P + (i << 30), n_rows=1, table_stride=5) for i in (0, 1024))      # refused: nothing is read
        tables_only = pool(pkg, k=None, v=None, n_pages=n_pages)
        assert K.b200_pages_update(C.byref(tables_only), C.byref(f), C.byref(t), None, P, P, P, P + 8192, 1 << 60, None) == ERR
        assert K.b200_pages_compact(C.byref(tables_only), C.byref(f), C.byref(t), P, P, P + 8192, 1 << 60, None) == ERR
        assert K.b200_pages_copy(C.byref(pool(pkg, n_pages=n_pages)), 1, P + 8192, 1 << 60, None) == ERR


def test_attention_and_store_refuse_what_overflows(K, pkg):
    """2^30 new tokens of one sequence and more (the store alone has no heads to count rows by), and rows of tables that no state can have."""
    pl = pool(pkg)
    ok = dict(q=P, q_type=1, nb_q_tok=512, nb_q_head=128, dst=P, nb_dst_tok=512, nb_dst_head=128, k_new=P, v_new=P, nb_new_tok=0, nb_new_head=128, layer=0, tables=P, table_stride=5, lens=P,
              q_start=P, n_tok=4, n_seq=1, n_head=4, max_new=2, max_len=20, causal=1, scale=0.1, workspace=P, workspace_bytes=1 << 60)
    for n in (1 << 30, (1 << 31) - 1):
        a = changed(pkg.PagedAttnArgs, ok, n_tok=n, max_new=n)
        assert K.b200_paged_store(C.byref(pl), C.byref(a), None) == ERR
    for stride in (1 << 31, 1 << 62):
        a = changed(pkg.PagedAttnArgs, ok, table_stride=stride)
        assert K.b200_paged_store(C.byref(pl), C.byref(a), None) == ERR and K.b200_paged_attn(C.byref(pl), C.byref(a), None) == ERR


def test_attention_and_store_refuse_an_unaligned_status(K, pkg):
    ok = dict(q=P, q_type=1, nb_q_tok=512, nb_q_head=128, dst=P, nb_dst_tok=512, nb_dst_head=128, k_new=P, v_new=P, nb_new_tok=256, nb_new_head=128, layer=0, tables=P, table_stride=5, lens=P,
              q_start=P, n_tok=4, n_seq=2, n_head=4, max_new=2, max_len=20, causal=1, scale=0.1, workspace=P, workspace_bytes=1 << 15, status=P + 2)
    for f in (K.b200_paged_attn, K.b200_paged_store):
        assert f(C.byref(pool(pkg)), C.byref(changed(pkg.PagedAttnArgs, ok)), None) == ERR


def test_pages_refuse_results_that_overlap_what_is_read(K, pkg):
    """Every CTA reads the inputs for itself while the results are written."""
    n = K.b200_pages_workspace(3, 10)
    at = dict(tables=P, lens=P + 1024, refs=P + 2048)
    to = dict(tables=P + 4096, lens=P + 5120, refs=P + 6144)
    rest = dict(parent=P + 512, keep=P + 600, n_new=P + 700, status=P + 800, remap=P + 3328, ws=P + 8192)

    def call(f=at, t=to, **kw):
        a = dict(rest, **kw)
        f, t = (pkg.PageState(n_rows=3, table_stride=5, **s) for s in (f, t))
        pl = pool(pkg)
        return (K.b200_pages_update(C.byref(pl), C.byref(f), C.byref(t), a["parent"], a["keep"], a["n_new"], a["status"], a["ws"], n, None),
                K.b200_pages_compact(C.byref(pl), C.byref(f), C.byref(t), a["remap"], a["status"], a["ws"], n, None))
    for name, size in (("tables", 60), ("lens", 12), ("refs", 40)):
        for other, at_other in list(at.items()) + [(k, v) for k, v in to.items() if k != name]:
            assert call(t=dict(to, **{name: at_other})) == (ERR, ERR), (name, other)
        assert call(status=to[name] + size - 4) == (ERR, ERR) and call(status=at[name]) == (ERR, ERR), name
        assert call(ws=to[name] // 16 * 16) == (ERR, ERR) and call(remap=to[name] + size - 4)[1] == ERR and call(remap=at[name])[1] == ERR, name
        for k in ("parent", "keep", "n_new"):
            assert call(**{k: to[name] + size - 4})[0] == ERR, (name, k)
    assert call(status=rest["keep"] + 4)[0] == ERR and call(status=rest["ws"]) == (ERR, ERR) and call(status=rest["remap"] + 8)[1] == ERR
