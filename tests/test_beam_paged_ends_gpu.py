"""Attention over the paged cache where weights are small, values infinite, steps have failed or are over; beam selection and page states at their ends.
Helpers and plain forms as in test_beam_paged_gpu.py."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as R
from test_beam_paged_gpu import K, Attn, Cache, Select, check_select, check_update, dev, p, run_update, stream  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def one_leader(K, pkg, seqs, Hkv, g, D, t, qt, ps, lead, at):
    """Every key of a sequence has the same score but the one at `at`, which lies `lead` nats above and has the value 0; all values have one sign."""
    x = Attn(K, pkg, np.random.default_rng(1), seqs, Hkv, g, D, t, qt, ps, store=False)
    x.q.zero_()
    x.q[..., 0] = 8.0
    x.c.view[0].zero_()
    x.c.view[1] = x.c.view[1].abs() + 1.0
    for i in range(len(seqs)):
        page, tok = int(x.tables[i, at // ps]), at % ps
        x.c.view[0, 0, page, tok, :, 0] = round(lead / (8.0 * x.scale) * 8) / 8      # exact in the pool's types
        x.c.view[1, 0, page, tok] = 0.0
    return x


FORMS = [
    # seqs, Hkv, g, D, ps, position of the leader: eight warps an item, four warps, the line, many rows (tcgen05, or 128 f32 rows a CTA), tcgen05 split
    ([(1, 400)], 2, 2, 64, 16, 40),
    ([(1, 400)] * 80, 2, 2, 64, 16, 40),
    ([(1, 40003)], 1, 2, 64, 16, 39000),
    ([(1, 9001), (1, 20002)], 2, 4, 128, 16, 8000),
    ([(200, 900)] * 4, 20, 1, 64, 16, 600),
    ([(200, 900)] * 4, 20, 1, 128, 16, 600),
    ([(300, 4000)], 2, 4, 128, 64, 3650),
    ([(300, 3000)], 10, 1, 64, 64, 2600),
]


@pytest.mark.parametrize("form", range(len(FORMS)))
@pytest.mark.parametrize("t,qt,lead", [("f16", "f16", 15), ("f16", "f16", 17), ("f16", "f32", 22), ("bf16", "bf16", 17), ("bf16", "f32", 22)])
def test_small_weights_beside_a_large_one(K, pkg, form, t, qt, lead):
    """What many keys far below the largest score add up to is there: exp(-17) = 2^-24.5 and, for f32 queries, exp(-22) = 2^-31.7 are below what f16
    holds with all its bits beside a weight of 1. Tolerances of Attn.check: roundings relative to every weight."""
    x = one_leader(K, pkg, *FORMS[form][:4], t, qt, FORMS[form][4], lead, FORMS[form][5])
    pool = x.c.view.clone()
    x.run()
    x.check(pool)


@pytest.mark.parametrize("form", range(len(FORMS)))
@pytest.mark.parametrize("t,qt", [("f16", "f16"), ("f16", "f32"), ("bf16", "bf16")])
def test_infinite_values_far_below_the_largest_score(K, pkg, form, t, qt):
    """A value that is attended to with a weight of exp(-200) leaves its dimension infinite or NaN, whichever warp, CTA or split has its key."""
    seqs, Hkv, g, D, ps, at = FORMS[form]
    x, y = (one_leader(K, pkg, seqs, Hkv, g, D, t, qt, ps, 200, at) for _ in range(2))
    for i in range(len(seqs)):
        x.c.view[1, 0, int(x.tables[i, 5 // ps]), 5 % ps, 0, 3] = float("inf")
        x.c.view[1, 0, int(x.tables[i, 5 // ps]), 5 % ps, Hkv - 1, 4] = float("nan")
    x.run()
    y.run()
    torch.cuda.synchronize()
    out, want = x.out[:x.n_tok].clone(), y.out[:x.n_tok]
    assert want.isfinite().all()
    assert not out[:, :g, 3].isfinite().any() and out[:, -g:, 4].isnan().all()
    out[:, :g, 3], out[:, -g:, 4] = want[:, :g, 3], want[:, -g:, 4]
    assert torch.equal(out, want) and torch.equal(x.lse, y.lse)


@pytest.mark.parametrize("V", [100, 9001, 51866])
@pytest.mark.parametrize("n_beam", [1, 5, 32])
def test_select_with_infinite_scores(K, pkg, V, n_beam):
    """A score of +inf makes a row's candidates equal: the lowest tokens that are allowed and have a logit above -inf."""
    rng = np.random.default_rng(V + n_beam)
    x = rng.standard_normal((3 * n_beam, V)).astype(np.float32)
    score = -rng.random(3 * n_beam).astype(np.float32)
    score[0] = np.inf                                      # one row beside ordinary ones
    score[n_beam:2 * n_beam] = np.inf                      # all of them, with logits that are none, and infinite ones
    x[n_beam, :min(50, V // 2)] = -np.inf
    x[n_beam, 3] = np.nan
    x[2 * n_beam - 1, V - 1] = np.inf
    score[2 * n_beam] = np.inf
    done = np.zeros(3 * n_beam, np.uint8)
    done[2 * n_beam] = 1
    banned = rng.random((1, V)) < 0.3
    for m in (None, banned):
        s = Select(K, pkg, torch.from_numpy(x).cuda(), score, done, m, 7, n_beam, 1, 1)
        s.run()
        with np.errstate(all="ignore"):
            check_select(s.got(), R.beam_select(x, score, done, m, 7, n_beam))


def test_steps_without_new_tokens(K, pkg):
    """Captured steps of many rows whose sequences are all finished: nothing is stored or written, and what follows may change the tables at once."""
    seqs = [(200, 260), (130, 130), (90, 400), (256, 300)]
    x = Attn(K, pkg, np.random.default_rng(2), seqs, 20, 1, 64, "f16", "f16", 16)
    first = x.c.view.clone()
    pool = x.want_pool(first)
    start, over = x.dstart.clone(), torch.zeros_like(x.dstart)
    next_lens, lens = torch.zeros_like(x.dlen), x.dlen.clone()
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            x.dstart.copy_(over)
            x.run()
            x.dlen.copy_(next_lens)
        for _ in range(20):
            x.dlen.copy_(lens)
            g.replay()
            x.run()
        st.synchronize()
        assert torch.equal(torch.nan_to_num(x.c.view, 3.0), torch.nan_to_num(first, 3.0)) and (x.out == 7).all() and (x.lse == 7).all()
        x.dlen.copy_(lens)
        x.dstart.copy_(start)
        x.run()
    torch.cuda.synchronize()
    x.check(pool)


@pytest.mark.parametrize("rows,n_pages", [(3, 12), (300, 40000)])
def test_update_refuses_entries_on_free_pages(K, pkg, rows, n_pages):
    """A used entry on a page that nobody holds would be handed out as new."""
    rng = np.random.default_rng(rows)
    c = Cache(pkg, rng, n_pages, 4, Hkv=1)
    tables = np.full((rows, 4), -1)
    tables[:, :2] = rng.permutation(n_pages)[:2 * rows].reshape(rows, 2)
    lens, before = np.full(rows, 7), c.view.clone()
    refs = np.bincount(tables[:, :2].ravel(), minlength=n_pages)
    for row, keep in ((0, 7), (rows - 1, 0), (rows // 2, 7)):
        free = refs.copy()
        free[tables[row, 1]] = 0
        k = lens.copy()
        k[row] = keep
        got, status, _ = run_update(K, pkg, c, tables, lens, free, None, k, np.ones(rows, int))
        check_update(c, before, got, status, (tables, lens, free, [], -1))
    got, status, _ = run_update(K, pkg, c, tables, lens, refs, None, lens, np.ones(rows, int))
    check_update(c, before, got, status, R.pages_update(tables, lens, refs, np.arange(rows), lens, np.ones(rows, int), 4))


@pytest.mark.parametrize("n_new,rows,heads,qt,t", [(1, 5, 4, "f16", "f16"), (1, 5, 4, "f32", "bf16"), (1, 300, 4, "bf16", "bf16"), (60, 4, 2, "f32", "f16"), (200, 5, 20, "f16", "f16"),
                                                   (200, 5, 20, "f32", "f16")])
def test_a_step_that_ran_out_of_pages_changes_no_page(K, pkg, n_new, rows, heads, qt, t):
    """The update leaves a copy of the state; attention and store with its status do nothing, so that the rows' last tokens stay what they were.
    With pages enough the same calls store and attend."""
    rng = np.random.default_rng(n_new)
    ps, D, n = 16, 64, 300
    used, more = R.ceil(n, ps), R.ceil(n + n_new, ps) - R.ceil(n, ps)
    width = used + more + 1
    for short in (True, False):
        n_pages = rows * (used + more) + (rows if more == 0 else -int(short))
        c = Cache(pkg, rng, n_pages, ps, heads, D, t)
        tables = np.full((rows, width), -1)
        tables[:, :used] = rng.permutation(n_pages)[:rows * used].reshape(rows, used)
        refs = np.bincount(tables[tables >= 0], minlength=n_pages)
        if short and more == 0:
            refs[refs == 0] = 1
            refs[tables[0, used - 1]] += 1                 # a holder besides: row 0 has to copy its last page, and none is free
        lens = np.full(rows, n)
        keep, new = lens.copy(), np.full(rows, n_new)
        frm, f = c.state(pkg, tables, lens, refs)
        to, s = c.state(pkg, np.zeros_like(tables), np.zeros_like(lens), np.zeros_like(refs))
        status = torch.full((2,), 55, dtype=torch.int32, device="cuda")
        m = K.b200_pages_workspace(rows, n_pages)
        ws = torch.empty(m, dtype=torch.uint8, device="cuda")
        dt = dict(f16=torch.float16, bf16=torch.bfloat16, f32=torch.float32)[qt]
        q, kn, vn = (torch.from_numpy(rng.standard_normal((rows * n_new, heads, D))).to(dt).cuda() for _ in range(3))
        out, lse = torch.full_like(q, 7.0), torch.full((rows * n_new, heads), 7.0, device="cuda")
        start, es = dev(np.arange(rows + 1) * n_new, np.int32), q.element_size()
        kd, nd = dev(keep, np.int32), dev(new, np.int32)
        a = pkg.PagedAttnArgs(q=p(q), q_type=dict(f32=0, f16=1, bf16=30)[qt], nb_q_tok=heads * D * es, nb_q_head=D * es, dst=p(out), nb_dst_tok=heads * D * es, nb_dst_head=D * es,
                              k_new=p(kn), v_new=p(vn), nb_new_tok=heads * D * es, nb_new_head=D * es, layer=0, tables=p(to["tables"]), table_stride=width, lens=p(to["lens"]),
                              q_start=p(start), n_tok=rows * n_new, n_seq=rows, n_head=heads, max_new=n_new, max_len=n + n_new, causal=1, scale=0.125, lse=p(lse), status=p(status))
        w = K.b200_paged_attn_workspace(C.byref(c.pool), C.byref(a))
        aws = torch.empty(max(w, 16), dtype=torch.uint8, device="cuda")
        a.workspace, a.workspace_bytes = p(aws), w
        before = c.view.clone()
        st = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):           # nothing between them looks at the status on the host
                assert K.b200_pages_update(C.byref(c.pool), C.byref(f), C.byref(s), None, p(kd), p(nd), p(status), p(ws), m, stream()) == 0
                assert K.b200_paged_store(C.byref(c.pool), C.byref(a), stream()) == 0
                assert K.b200_paged_attn(C.byref(c.pool), C.byref(a), stream()) == 0
            g.replay()
            st.synchronize()
        if short:
            assert status.tolist() == [1, 0] and torch.equal(c.view, before)
            assert (out == 7).all() and (lse == 7).all()
            continue
        assert status.tolist()[0] == 0
        table = to["tables"].cpu().numpy()
        for i in range(rows):
            for j, x in enumerate((kn, vn)):
                pos = n + np.arange(n_new)
                assert torch.equal(c.view[j, 0][torch.from_numpy(table[i, pos // ps]).long().cuda(), torch.from_numpy(pos % ps).cuda()],
                                   x[i * n_new:(i + 1) * n_new].to(c.view.dtype))
        assert not (out == 7).all() and lse.isfinite().all() and not (lse == 7).any()


def test_beams_that_run_out_of_candidates(K, pkg):
    """A step over several sequences in which the second has fewer candidates than beams: the beams without one (parent -1) give their pages back, take
    nothing from another sequence, and come back when a later selection gives them a parent."""
    rng = np.random.default_rng(4)
    n_seq, nb, V, ps, width, n_pages = 3, 4, 50, 4, 6, 80
    rows = n_seq * nb
    c = Cache(pkg, rng, n_pages, ps, Hkv=1)
    tables = np.full((rows, width), -1)
    tables[:, :3] = rng.permutation(n_pages)[:rows * 3].reshape(rows, 3)
    lens = np.repeat([9, 10, 11], nb)
    refs = np.bincount(tables[tables >= 0], minlength=n_pages)
    score = -rng.random(rows).astype(np.float32)
    x = rng.standard_normal((2, rows, V)).astype(np.float32)
    x[0, nb:2 * nb] = -np.inf
    x[0, nb + 2, 5] = 1.0                                  # one candidate in the second sequence
    score[0:nb] = -np.inf                                  # and none at all in the first
    done = np.zeros(rows, np.uint8)
    for step in range(2):
        s = Select(K, pkg, torch.from_numpy(x[step]).cuda(), score, done, None, 3, nb)
        s.run()
        got = s.got()
        check_select(got, R.beam_select(x[step], score, done, None, 3, nb))
        parent, score, done = got["parent"], got["score"], got["done"]
        own, none = np.arange(rows), parent < 0
        row_parent = np.where(none, own, own // nb * nb + parent)
        keep = np.where(none, 0, lens[row_parent])
        new = np.where(none | (done != 0), 0, 1)
        before = c.view.clone()
        want = R.pages_update(tables, lens, refs, row_parent, keep, new, ps)
        up, status, _ = run_update(K, pkg, c, tables, lens, refs, row_parent, keep, new)
        assert status[0] == 0
        check_update(c, before, up, status, want)
        old = {i // nb: set(tables[i // nb * nb:(i // nb + 1) * nb].ravel()) for i in range(rows)}
        for i in range(rows):
            other = set().union(*(old[q] for q in old if q != i // nb)) - {-1}
            assert not other & set(up["tables"][i])
        assert (up["lens"][none] == 0).all() and (up["tables"][none] == -1).all()
        tables, lens, refs = (up[k].astype(int) for k in ("tables", "lens", "refs"))
    assert none[:nb].all() and (refs == np.bincount(tables[tables >= 0], minlength=n_pages)).all()


def test_the_wait_status_waits_for_every_stream(K, pkg):
    """Streams that do not wait for the default stream are waited for as well."""
    st = torch.cuda.Stream()
    x = Attn(K, pkg, np.random.default_rng(0), [(300, 400)], 1, 1, 128, "f16", "f16", 16)
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        torch.cuda._sleep(200_000_000)                     # about a tenth of a second
        x.run()
    assert K.b200_paged_attn_status() == 0 and st.query()
