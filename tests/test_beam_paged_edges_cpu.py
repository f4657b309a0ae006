"""More refusals of the beam-search and paged-cache entry points; helpers as in test_beam_paged_cpu.py."""
import ctypes as C

from test_beam_paged_cpu import ERR, K, P, changed, pool  # noqa: F401


def test_select_and_reorder_refuse_unaligned_words(K, pkg):
    ok = dict(logits=P, type=0, nb_row=400, n_vocab=100, n_seq=2, n_beam=3, score=P, eos=1, score_out=P, token_out=P, parent_out=P, done_out=P, workspace=P,
              workspace_bytes=K.b200_beam_select_workspace(2, 3, 100))
    for name in ("score", "banned", "score_out", "token_out", "parent_out"):
        assert K.b200_beam_select(C.byref(changed(pkg.BeamSelectArgs, ok, **{name: P + 2})), None) == ERR, name
    b = (pkg.BeamBlock * 1)(pkg.BeamBlock(base=P, n_outer=1, nb_outer=0, nb_row=64, row_bytes=60))
    assert K.b200_beam_reorder(b, 1, P + 1, 2, 3, None) == ERR


def test_pages_refuse_unaligned_words_and_huge_pages(K, pkg):
    n = K.b200_pages_workspace(3, 10)
    ok_f = dict(tables=P, lens=P + 1024, refs=P + 2048, n_rows=3, table_stride=5)
    ok_t = dict(ok_f, tables=P + 4096, lens=P + 5120, refs=P + 6144)

    def update(pl=None, f={}, t={}, parent=None, keep=P, new=P, status=P):
        return K.b200_pages_update(C.byref(pl or pool(pkg)), C.byref(changed(pkg.PageState, ok_f, **f)), C.byref(changed(pkg.PageState, ok_t, **t)), parent, keep, new, status, P + 8192, n, None)
    for kw in (dict(f=dict(tables=P + 1)), dict(f=dict(lens=P + 1022)), dict(t=dict(refs=P + 6147)), dict(parent=P + 2), dict(keep=P + 2), dict(new=P + 1), dict(status=P + 3)):
        assert update(**kw) == ERR, kw
    for kw in (dict(remap=P + 2), dict(status=P + 2)):
        a = dict(dict(remap=P, status=P), **kw)
        assert K.b200_pages_compact(C.byref(pool(pkg)), C.byref(changed(pkg.PageState, ok_f)), C.byref(changed(pkg.PageState, ok_t)), a["remap"], a["status"], P + 8192, n, None) == ERR, kw
    row = 256                                              # a page of 2^20 tokens of 256 heads: 64 GB
    huge = pool(pkg, page_size=1 << 20, n_head_kv=256, head_dim=128, nb_head=row, nb_tok=256 * row, nb_page=256 * row << 20, nb_layer=0)
    assert update(huge) == ERR
    assert K.b200_pages_copy(C.byref(huge), 3, P, n, None) == ERR


def test_attention_refuses_unaligned_words_and_too_many_rows(K, pkg):
    ok = dict(q=P, q_type=1, nb_q_tok=512, nb_q_head=128, dst=P, nb_dst_tok=512, nb_dst_head=128, k_new=P, v_new=P, nb_new_tok=256, nb_new_head=128, layer=0, tables=P, table_stride=5, lens=P,
              q_start=P, n_tok=4, n_seq=2, n_head=4, max_new=2, max_len=20, causal=1, scale=0.1, workspace=P, workspace_bytes=1 << 15)
    for name in ("tables", "lens", "q_start"):
        for f in (K.b200_paged_attn, K.b200_paged_store):
            assert f(C.byref(pool(pkg)), C.byref(changed(pkg.PagedAttnArgs, ok, **{name: P + 2})), None) == ERR, name
    for kw in (dict(lse=P + 2), dict(n_tok=1 << 30, max_new=1 << 30, workspace_bytes=1 << 60), dict(n_head=4096, n_tok=1 << 20, max_new=1 << 30, workspace_bytes=1 << 60)):
        assert K.b200_paged_attn(C.byref(pool(pkg)), C.byref(changed(pkg.PagedAttnArgs, ok, **kw)), None) == ERR, kw
    for scale in (3e38, -3e38, float("inf"), float("nan")):        # times log2(e) no float
        assert K.b200_paged_attn(C.byref(pool(pkg)), C.byref(changed(pkg.PagedAttnArgs, ok, scale=scale)), None) == ERR


def test_attention_workspace_is_bounded(K, pkg):
    import random
    rng = random.Random(1)
    most = 0
    for _ in range(20000):
        d, kv = rng.choice([64, 128]), rng.choice([1, 2, 4, 6, 8, 12, 20, 32])
        pl = pool(pkg, head_dim=d, n_head_kv=kv, nb_head=2 * d, nb_tok=2 * d * kv, nb_page=8 * d * kv, page_size=4)
        new, seqs = int(2 ** rng.uniform(0, 13)), int(2 ** rng.uniform(0, 9))
        a = pkg.PagedAttnArgs(q_type=rng.choice([0, 1]), n_tok=new * seqs, n_seq=seqs, n_head=kv * rng.choice([1, 2, 4, 8]), max_new=new, max_len=int(2 ** rng.uniform(0, 20)))
        most = max(most, K.b200_paged_attn_workspace(C.byref(pl), C.byref(a)))
    assert 0 < most <= 21_000_000
