"""Refusals of the beam-search and paged-cache entry points: arguments are checked before anything is launched, so bad ones come back
as error codes on a machine without a GPU as well."""
import ctypes as C

import numpy as np
import pytest

ERR = 10001
BUF = np.zeros(1 << 16, np.uint8)
P = BUF.ctypes.data + (-BUF.ctypes.data % 256)


@pytest.fixture(scope="module")
def K(pkg):
    return pkg.kernels_lib()


def changed(cls, ok, **kw):
    return cls(**dict(ok, **kw))


def test_select_refuses(K, pkg):
    ok = dict(logits=P, type=0, nb_row=400, n_vocab=100, n_seq=2, n_beam=3, score=P, eos=1, score_out=P, token_out=P, parent_out=P, done_out=P, workspace=P,
              workspace_bytes=K.b200_beam_select_workspace(2, 3, 100))
    assert K.b200_beam_select_workspace(2, 3, 100) > 0
    for kw in (dict(logits=None), dict(logits=P + 2), dict(type=8), dict(nb_row=396), dict(nb_row=402), dict(n_vocab=0), dict(n_beam=0), dict(n_beam=33), dict(n_seq=-1),
               dict(score=None), dict(score_out=None), dict(token_out=None), dict(parent_out=None), dict(done_out=None), dict(workspace=None), dict(workspace=P + 4),
               dict(workspace_bytes=ok["workspace_bytes"] - 1), dict(banned_stride=-1), dict(n_vocab=1 << 31, nb_row=1 << 40), dict(n_vocab=1 << 27, n_beam=32, nb_row=1 << 30)):
        assert K.b200_beam_select(C.byref(changed(pkg.BeamSelectArgs, ok, **kw)), None) == ERR, kw
    assert K.b200_beam_select(None, None) == ERR
    assert K.b200_beam_select(C.byref(changed(pkg.BeamSelectArgs, ok, n_seq=0)), None) == 0          # nothing to do
    assert K.b200_beam_select_workspace(1, 33, 100) == 0 and K.b200_beam_select_workspace(1, 1, 0) == 0


def test_reorder_refuses(K, pkg):
    ok = dict(base=P, n_outer=2, nb_outer=6 * 64, nb_row=64, row_bytes=60)

    def call(n=1, parent=P, n_seq=2, n_beam=3, **kw):
        b = (pkg.BeamBlock * 9)(*[changed(pkg.BeamBlock, ok, **kw)] * 9)
        return K.b200_beam_reorder(b, n, parent, n_seq, n_beam, None)
    for kw in (dict(base=None), dict(nb_row=59), dict(n_outer=-1), dict(row_bytes=-1), dict(nb_outer=100), dict(nb_outer=-384), dict(n=9), dict(n=-1), dict(parent=None), dict(n_seq=-1),
               dict(n_beam=0), dict(n_beam=33), dict(row_bytes=1 << 41, nb_row=1 << 41)):
        assert call(**kw) == ERR, kw
    assert K.b200_beam_reorder(None, 1, P, 1, 2, None) == ERR
    for kw in (dict(n=0), dict(n_seq=0), dict(row_bytes=0), dict(n_outer=0), dict(n_beam=1)):
        assert call(**kw) == 0, kw                         # nothing to move


def pool(pkg, **kw):
    return changed(pkg.PagePool, dict(k=P, v=P, type=1, n_layer=1, n_pages=10, page_size=4, n_head_kv=2, head_dim=64, nb_layer=10240, nb_page=1024, nb_tok=256, nb_head=128), **kw)


BAD_POOLS = [dict(v=None), dict(k=P + 8), dict(type=0), dict(type=8), dict(n_layer=0), dict(n_pages=0), dict(page_size=0), dict(n_head_kv=0), dict(head_dim=80), dict(nb_page=1000),
             dict(nb_tok=8), dict(nb_head=64), dict(nb_head=-128), dict(n_layer=2, nb_layer=10248)]


def test_pages_refuse(K, pkg):
    n = K.b200_pages_workspace(3, 10)
    assert n > 0 and K.b200_pages_workspace(-1, 10) == 0 and K.b200_pages_workspace(1, 0) == 0 and K.b200_pages_workspace(8193, 10) == 0
    ok_f = dict(tables=P, lens=P + 1024, refs=P + 2048, n_rows=3, table_stride=5)
    ok_t = dict(ok_f, tables=P + 4096, lens=P + 5120, refs=P + 6144)

    def update(pl=None, f={}, t={}, keep=P, new=P, status=P, ws=P + 8192, ws_n=n):
        return K.b200_pages_update(C.byref(pl or pool(pkg)), C.byref(changed(pkg.PageState, ok_f, **f)), C.byref(changed(pkg.PageState, ok_t, **t)), None, keep, new, status, ws, ws_n, None)

    def compact(pl=None, f={}, t={}, remap=P, status=P, ws=P + 8192, ws_n=n):
        return K.b200_pages_compact(C.byref(pl or pool(pkg)), C.byref(changed(pkg.PageState, ok_f, **f)), C.byref(changed(pkg.PageState, ok_t, **t)), remap, status, ws, ws_n, None)
    for kw in BAD_POOLS:
        assert update(pool(pkg, **kw)) == ERR and compact(pool(pkg, **kw)) == ERR, kw
        assert K.b200_pages_copy(C.byref(pool(pkg, **kw)), 3, P + 8192, 1 << 14, None) == ERR, kw
    for call in (update, compact):
        for f in (dict(tables=None), dict(lens=None), dict(refs=None), dict(n_rows=-1), dict(n_rows=8193), dict(n_rows=2), dict(table_stride=0), dict(table_stride=6),
                  dict(tables=P + 4096 + 8), dict(refs=P + 6144), dict(lens=P + 5124)):
            assert call(f=f) == ERR, f
        assert call(f=dict(table_stride=1 << 29), t=dict(table_stride=1 << 29)) == ERR
        for kw in (dict(status=None), dict(ws=None), dict(ws=P + 8196), dict(ws_n=n - 1)):
            assert call(**kw) == ERR, kw
    assert update(keep=None) == ERR and update(new=None) == ERR and compact(remap=None) == ERR
    assert K.b200_pages_copy(C.byref(pool(pkg)), 3, P, n - 1, None) == ERR and K.b200_pages_copy(C.byref(pool(pkg)), -1, P, n, None) == ERR
    assert K.b200_pages_copy(C.byref(pool(pkg)), 3, None, n, None) == ERR


def test_attention_refuses(K, pkg):
    ok = dict(q=P, q_type=1, nb_q_tok=512, nb_q_head=128, dst=P, nb_dst_tok=512, nb_dst_head=128, k_new=P, v_new=P, nb_new_tok=256, nb_new_head=128, layer=0, tables=P, table_stride=5, lens=P,
              q_start=P, n_tok=4, n_seq=2, n_head=4, max_new=2, max_len=20, causal=1, scale=0.1, workspace=P, workspace_bytes=1 << 15)

    def call(f, pl=None, **kw):
        return f(C.byref(pl or pool(pkg)), C.byref(changed(pkg.PagedAttnArgs, ok, **kw)), None)
    for kw in BAD_POOLS:
        assert call(K.b200_paged_attn, pool(pkg, **kw)) == ERR and call(K.b200_paged_store, pool(pkg, **kw)) == ERR, kw
    both = (dict(layer=1), dict(layer=-1), dict(n_seq=-1), dict(n_tok=-1), dict(max_new=-1), dict(max_len=-1), dict(max_len=1 << 30), dict(q_type=30), dict(q_type=8), dict(tables=None),
            dict(table_stride=0), dict(lens=None), dict(q_start=None), dict(k_new=None), dict(v_new=None), dict(k_new=P + 8), dict(nb_new_tok=250), dict(nb_new_head=-128), dict(n_seq=65536))
    for kw in both:
        assert call(K.b200_paged_attn, **kw) == ERR and call(K.b200_paged_store, **kw) == ERR, kw
    for kw in (dict(q=None), dict(dst=None), dict(q=P + 2), dict(dst=P + 8), dict(n_head=3), dict(n_head=0), dict(nb_q_tok=520), dict(nb_dst_tok=64), dict(nb_dst_head=64), dict(nb_q_head=-128),
               dict(scale=float("nan")), dict(scale=float("inf"))):
        assert call(K.b200_paged_attn, **kw) == ERR, kw
    assert call(K.b200_paged_store, k_new=None, v_new=None) == ERR
    for kw in (dict(n_seq=0), dict(n_tok=0), dict(max_new=0)):
        assert call(K.b200_paged_attn, **kw) == 0 and call(K.b200_paged_store, **kw) == 0, kw
    assert K.b200_paged_attn(None, None, None) == ERR
    need = K.b200_paged_attn_workspace(C.byref(pool(pkg)), C.byref(changed(pkg.PagedAttnArgs, ok, max_len=4000, n_tok=1, n_seq=1)))
    assert need > 0 and call(K.b200_paged_attn, max_len=4000, n_tok=1, n_seq=1, workspace_bytes=need - 1) == ERR
    assert call(K.b200_paged_attn, max_len=4000, n_tok=1, n_seq=1, workspace=None) == ERR and call(K.b200_paged_attn, max_len=4000, n_tok=1, n_seq=1, workspace=P + 8) == ERR
