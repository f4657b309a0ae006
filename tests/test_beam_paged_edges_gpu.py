"""Beam selection, the paged cache and attention over it where sizes, offsets and concurrency are at their ends; helpers and plain forms as in
test_beam_paged_gpu.py."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as R
import test_beam_paged_gpu as B
from test_beam_paged_gpu import K, Attn, Cache, Select, check_select, check_update, dev, p, random_state, run_update, stream  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


class FarCache(Cache):
    """Pages 800 MB apart: from the sixth on, offsets inside a layer pass 32 bits."""

    def __init__(self, pkg, rng, n_pages, ps, Hkv=2, D=64, t="f16", n_layer=1, layout="tok", gap=0):
        near = Cache(pkg, rng, n_pages, ps, Hkv, D, t, n_layer, layout, 0)
        self.__dict__.update(near.__dict__)
        page = 400 << 20                                   # elements
        self.buf = torch.empty((2, n_layer, n_pages, page), dtype=B.DT[t], device="cuda")
        self.view = self.buf[..., : ps * Hkv * D].unflatten(-1, (ps, Hkv, D) if layout == "tok" else (Hkv, ps, D))
        if layout != "tok":
            self.view = self.view.transpose(3, 4)
        self.view.copy_(near.view)
        self.pool.k, self.pool.v = p(self.buf[0]), p(self.buf[1])
        self.pool.nb_page, self.pool.nb_layer = page * 2, n_pages * page * 2


@pytest.fixture
def far(monkeypatch):
    monkeypatch.setattr(B, "Cache", FarCache)
    yield FarCache
    torch.cuda.empty_cache()


@pytest.mark.parametrize("seqs,g,D,ps,qt", [([(1, 200), (1, 70)], 4, 128, 40, "f32"), ([(200, 230), (1, 40)], 1, 64, 64, "f16"), ([(150, 260)], 2, 128, 48, "f16"),
                                            ([(20, 130), (0, 0), (3, 100)], 2, 64, 48, "f32")])
def test_attention_of_pages_far_apart(K, pkg, far, seqs, g, D, ps, qt):
    x = Attn(K, pkg, np.random.default_rng(len(seqs)), seqs, 2, g, D, "f16", qt, ps)
    assert x.c.n_pages * x.c.pool.nb_page > 1 << 32
    pool = x.want_pool(x.c.view)
    x.run()
    x.check(pool)


def test_update_and_compact_of_pages_far_apart(K, pkg, far):
    rng = np.random.default_rng(4)
    c = FarCache(pkg, rng, 12, 8, layout="head")
    tables, lens, refs = np.array([[9, 3, -1], [9, 11, -1]]), np.array([13, 12]), np.bincount([9, 3, 9, 11], minlength=12)
    before = c.view.clone()
    got, status, _ = run_update(K, pkg, c, tables, lens, refs, [1, 1], [12, 12], [1, 5])
    check_update(c, before, got, status, R.pages_update(tables, lens, refs, [1, 1], [12, 12], [1, 5], 8))
    before = c.view.clone()
    frm, f = c.state(pkg, got["tables"], got["lens"], got["refs"])
    to, t = c.state(pkg, np.zeros_like(tables), np.zeros_like(lens), np.zeros_like(refs))
    status, remap = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in (2, 12))
    n = K.b200_pages_workspace(2, 12)
    ws = torch.full((n,), 255, dtype=torch.uint8, device="cuda")
    assert K.b200_pages_compact(C.byref(c.pool), C.byref(f), C.byref(t), p(remap), p(status), p(ws), n, stream()) == 0
    torch.cuda.synchronize()
    moves = R.pages_compact(got["tables"], got["lens"], got["refs"], 8)[4]
    assert status.tolist() == [0, len(moves)] and len(moves) > 0
    for a, b in moves:
        assert torch.equal(c.view[:, :, b], before[:, :, a])


@pytest.mark.parametrize("n_new,length,qt", [(1, 200001, "f32"), (1, 131072, "f16"), (70, 60003, "f16")])
def test_attention_over_long_contexts(K, pkg, n_new, length, qt):
    x = Attn(K, pkg, np.random.default_rng(length), [(n_new, length), (1, 3)], 1, 2, 64, "f16", qt, 16)
    pool = x.want_pool(x.c.view)
    x.run()
    x.check(pool)


@pytest.mark.parametrize("ps", [3, 24, 48, 256, 512])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("qt", ["f16", "f32"])
def test_attention_page_sizes(K, pkg, ps, D, qt):
    """Pages larger than a block of keys, and pages that end inside one."""
    x = Attn(K, pkg, np.random.default_rng(ps), [(150, 700), (1, 513), (90, 90), (256, 256)], 2, 1, D, "f16", qt, ps)
    pool = x.want_pool(x.c.view)
    x.run()
    x.check(pool)


@pytest.mark.parametrize("n_new", [1, 3, 16, 17, 64, 65, 129])
@pytest.mark.parametrize("qt", ["f16", "f32"])
def test_more_new_tokens_than_length(K, pkg, n_new, qt):
    """The first queries stand before the sequence's begin: zeros, lse -inf, nothing stored."""
    x = Attn(K, pkg, np.random.default_rng(n_new), [(n_new, n_new // 2), (n_new, 0), (n_new, n_new + 1)], 2, 1, 64, "f16", qt, 8)
    pool = x.want_pool(x.c.view)
    x.run()
    x.check(pool)
    first = n_new - n_new // 2
    assert (x.out[:first] == 0).all() and (x.out[n_new:2 * n_new] == 0).all() and (x.lse[n_new:2 * n_new] == -np.inf).all()


def test_attention_finite_but_huge_scores(K, pkg):
    """Scores near the end of f32's range and weights that all but one key lose; q . k of opposite signs."""
    for n_new in (2, 100):
        x = Attn(K, pkg, np.random.default_rng(n_new), [(n_new, n_new + 40)], 1, 1, 64, "bf16", "bf16", 16, scale=1.0)
        x.q.mul_(3e17); x.kn.mul_(3e17)                    # the new keys only: scores of +-1e36 beside the past's +-1e18
        pool = x.want_pool(x.c.view)
        x.run()
        torch.cuda.synchronize()
        k, v = (pool[j, 0].double().cpu().numpy()[x.tables[0, np.arange(n_new + 40) // 16], np.arange(n_new + 40) % 16] for j in (0, 1))
        out, _, _, _ = R.attention(x.q.double().cpu().numpy(), k, v, n_new, n_new + 40, 1.0, 1)
        assert np.all(np.abs(x.out[:n_new].double().cpu().numpy() - out) <= 2.0 ** -8 * np.abs(out) + 1e-30)


@pytest.mark.parametrize("layout", ["tok", "head"])
@pytest.mark.parametrize("t,qt", [("f16", "f32"), ("bf16", "bf16")])
def test_store_alone(K, pkg, layout, t, qt):
    """The store by itself, then attention over what it stored: the bits of attention that stores."""
    seqs = [(5, 70), (0, 3), (40, 40), (1, 17)]
    x = Attn(K, pkg, np.random.default_rng(1), seqs, 2, 2, 64, t, qt, 16, layout=layout)
    y = Attn(K, pkg, np.random.default_rng(1), seqs, 2, 2, 64, t, qt, 16, layout=layout)
    pool = x.want_pool(x.c.view)
    assert K.b200_paged_store(C.byref(x.c.pool), C.byref(x.a), stream()) == 0
    torch.cuda.synchronize()
    assert torch.equal(torch.nan_to_num(x.c.view, 3.0), torch.nan_to_num(pool, 3.0)) and (x.out == 7).all()
    x.a.k_new = x.a.v_new = None
    x.run()
    y.run()
    x.check(pool)
    assert torch.equal(x.out, y.out) and torch.equal(x.lse, y.lse)


def test_calls_at_once_on_two_streams(K, pkg):
    """Selections, attention of single tokens and of chunks on two streams, each with its own scratch memory: the bits of serial calls."""
    rng = np.random.default_rng(3)

    def make(seed):
        r = np.random.default_rng(seed)
        logits = torch.from_numpy(r.standard_normal((200, 9001)).astype(np.float32)).cuda()
        return [Select(K, pkg, logits, -r.random(200).astype(np.float32), None, None, 3, 5),
                Attn(K, pkg, r, [(1, int(n)) for n in r.integers(1, 4000, 24)], 2, 4, 128, "bf16", "bf16", 16),
                Attn(K, pkg, r, [(200, 1500), (70, 600)], 2, 4, 128, "bf16", "bf16", 16),
                Attn(K, pkg, r, [(200, 900)] * 3, 4, 1, 64, "f16", "f16", 16)]

    def outputs(ops):
        return [o.got() if isinstance(o, Select) else (o.out.clone(), o.lse.clone()) for o in ops]

    def same(a, b):
        return all(np.array_equal(a[k], b[k]) for k in a) if isinstance(a, dict) else torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    sides = [make(1), make(2)]
    want = []
    for ops in sides:
        for o in ops:
            o.run()
        torch.cuda.synchronize()
        want.append(outputs(ops))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for i in rng.permutation(8):
            with torch.cuda.stream(streams[i % 2]):
                sides[i % 2][i // 2].run()
    torch.cuda.synchronize()
    for ops, w in zip(sides, want):
        assert all(same(a, b) for a, b in zip(outputs(ops), w))


def test_a_step_of_the_cache_captured_and_replayed(K, pkg):
    """reorder + update + attention + compact in one graph, replayed with other parents and lengths: what plain calls give."""
    rng = np.random.default_rng(8)
    n_seq, nb, ps, width, n_pages = 3, 4, 8, 8, 120
    rows = n_seq * nb
    tables, lens, refs = random_state(rng, n_seq, nb, ps, 40, n_pages, width)
    results = []
    plans = [(np.arange(rows) // nb * nb + r.integers(0, nb, rows), r.integers(0, 2, rows)) for r in (np.random.default_rng(s) for s in (1, 2))]
    st = torch.cuda.Stream()
    for captured in (False, True):
        r = np.random.default_rng(5)
        c = Cache(pkg, r, n_pages, ps, 2, 64, "f16")
        clean = c.buf.clone()
        s0, f = c.state(pkg, tables, lens, refs)
        s1, t = c.state(pkg, tables, lens, refs)
        s2, u = c.state(pkg, tables, lens, refs)
        hist0 = torch.from_numpy(r.integers(0, 1000, (rows, 40))).int().cuda()
        hist, par, keep, new, status = hist0.clone(), *(torch.zeros(rows, dtype=torch.int32, device="cuda") for _ in range(3)), torch.zeros(4, dtype=torch.int32, device="cuda")
        remap = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
        local = torch.zeros(rows, dtype=torch.int32, device="cuda")
        n = K.b200_pages_workspace(rows, n_pages)
        ws = torch.empty(n, dtype=torch.uint8, device="cuda")
        q = torch.from_numpy(r.standard_normal((rows, 4, 64))).half().cuda()
        out, start = torch.zeros_like(q), dev(np.arange(rows + 1, dtype=np.int32))
        a = pkg.PagedAttnArgs(q=p(q), q_type=1, nb_q_tok=512, nb_q_head=128, dst=p(out), nb_dst_tok=512, nb_dst_head=128, layer=0, tables=p(s1["tables"]), table_stride=width,
                              lens=p(s1["lens"]), q_start=p(start), n_tok=rows, n_seq=rows, n_head=4, max_new=1, max_len=width * ps, causal=1, scale=0.125)
        m = K.b200_paged_attn_workspace(C.byref(c.pool), C.byref(a))
        aws = torch.empty(max(m, 16), dtype=torch.uint8, device="cuda")
        a.workspace, a.workspace_bytes = p(aws), m
        blk = (pkg.BeamBlock * 1)(pkg.BeamBlock(base=p(hist), n_outer=1, nb_outer=0, nb_row=160, row_bytes=160))

        def step(s):
            assert K.b200_beam_reorder(blk, 1, p(local), n_seq, nb, s) == 0
            assert K.b200_pages_update(C.byref(c.pool), C.byref(f), C.byref(t), p(par), p(keep), p(new), p(status), p(ws), n, s) == 0
            assert K.b200_paged_attn(C.byref(c.pool), C.byref(a), s) == 0
            assert K.b200_pages_compact(C.byref(c.pool), C.byref(t), C.byref(u), p(remap), p(status) + 8, p(ws), n, s) == 0
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            g = torch.cuda.CUDAGraph()
            if captured:
                with torch.cuda.graph(g, stream=st):
                    step(st.cuda_stream)
            for parent, grow in plans:
                c.buf.copy_(clean); hist.copy_(hist0)
                par.copy_(torch.from_numpy(parent)); local.copy_(torch.from_numpy(parent % nb)); keep.copy_(torch.from_numpy(lens[parent])); new.copy_(torch.from_numpy(grow))
                if captured:
                    g.replay()
                else:
                    step(st.cuda_stream)
                st.synchronize()
                results.append([x.clone() for x in (c.buf, hist, out, status, remap, *s1.values(), *s2.values())])
                assert status.tolist()[0] == 0 and status.tolist()[2] == 0
    for i in (0, 1):
        assert all(torch.equal(x, y) for x, y in zip(results[i], results[i + 2]))
    assert not torch.equal(results[0][1], results[1][1])


def test_copies_of_a_workspace_that_was_never_used(K, pkg):
    """Numbers that are no pages are passed over."""
    c = Cache(pkg, np.random.default_rng(0), 20, 8, layout="head")
    before = c.buf.clone()
    n = K.b200_pages_workspace(4, 20)
    for fill in (255, 127, 128):
        ws = torch.full((n,), fill, dtype=torch.uint8, device="cuda")
        assert K.b200_pages_copy(C.byref(c.pool), 4, p(ws), n, stream()) == 0
    torch.cuda.synchronize()
    assert torch.equal(c.buf, before)


@pytest.mark.parametrize("groups,beams,width", [(2048, 4, 4), (8192, 1, 5), (1, 8, 20000)])
def test_update_and_compact_of_the_largest_states(K, pkg, groups, beams, width):
    rng = np.random.default_rng(width)
    rows, ps = groups * beams, 1
    n_pages = rows * (width + 1) + 5
    c = Cache(pkg, rng, n_pages, ps, Hkv=1)
    tables, lens, refs = random_state(rng, groups, beams, ps, width - 1, n_pages, width)
    parent = np.arange(rows) // beams * beams + rng.integers(0, beams, rows)
    keep, new = lens[parent].copy(), np.ones(rows, int)
    cut = rng.random(rows) < 0.4
    keep[cut] = (keep[cut] * rng.random(cut.sum())).astype(int)
    before = c.view.clone()
    got, status, _ = run_update(K, pkg, c, tables, lens, refs, parent, keep, new)
    check_update(c, before, got, status, R.pages_update(tables, lens, refs, parent, keep, new, ps))
    frm, f = c.state(pkg, got["tables"], got["lens"], got["refs"])
    to, t = c.state(pkg, np.zeros_like(tables), np.zeros_like(lens), np.zeros_like(refs))
    status, remap = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in (2, n_pages))
    n = K.b200_pages_workspace(rows, n_pages)
    ws = torch.full((n,), 255, dtype=torch.uint8, device="cuda")
    assert K.b200_pages_compact(C.byref(c.pool), C.byref(f), C.byref(t), p(remap), p(status), p(ws), n, stream()) == 0
    torch.cuda.synchronize()
    wt, wl, wr, wm, moves = R.pages_compact(got["tables"], got["lens"], got["refs"], ps)
    assert status.tolist() == [0, len(moves)] and np.array_equal(remap.cpu().numpy(), wm)
    assert np.array_equal(to["tables"].cpu().numpy(), wt) and np.array_equal(to["lens"].cpu().numpy(), wl) and np.array_equal(to["refs"].cpu().numpy(), wr)


@pytest.mark.parametrize("n_seq,n_beam,V", [(1, 32, 51866), (12, 5, 51866), (3, 32, 20000), (1, 32, 400000)])
@pytest.mark.parametrize("ties", [False, True])
def test_select_many_candidates(K, pkg, n_seq, n_beam, V, ties):
    """More lists than a thread holds, and whole slices of equal logits."""
    rng = np.random.default_rng(V + n_beam)
    x = rng.standard_normal((n_seq * n_beam, V)).astype(np.float32)
    score = -rng.random(n_seq * n_beam).astype(np.float32)
    if ties:
        x = np.round(x)                                    # a few values only
        x[::2] = 0.25
        score[:] = -1.0
    s = Select(K, pkg, torch.from_numpy(x).cuda(), score, None, None, 2, n_beam)
    s.run()
    want = R.beam_select(x.astype(np.float64), score, None, None, 2, n_beam)
    got = s.got()
    if not ties:
        check_select(got, want)
        return
    # rows of the same score and the same logits are equal to the last bit, others may change places within the error of their sums
    assert np.all(np.abs(got["score"] - want["score"]) <= 5e-6 + np.abs(want["score"]) * 2.0 ** -24)
    lp = x - x.max(1, keepdims=True)
    lp = lp.astype(np.float64) - np.log(np.exp(lp.astype(np.float64)).sum(1, keepdims=True)) - 1.0
    for q in range(n_seq):
        picked = set()
        for r in range(q * n_beam, (q + 1) * n_beam):
            b, t = int(got["parent"][r]), int(got["token"][r])
            assert abs(lp[q * n_beam + b, t] - got["score"][r]) <= 5e-6 + abs(got["score"][r]) * 2.0 ** -24 and (b, t) not in picked
            # the lowest indices of a row's equal logits come first
            same = np.flatnonzero(x[q * n_beam + b, :t] == x[q * n_beam + b, t])
            assert all((b, int(u)) in picked for u in same)
            picked.add((b, t))


WIDE = [([(300, 700)] * 3 + [(0, 5), (129, 129), (65, 64), (1, 40)], 12, 1, 64, 16), ([(80, 300), (0, 0), (257, 270)], 8, 6, 128, 24), ([(100, 90)] * 8, 20, 1, 64, 7)]


@pytest.mark.parametrize("shape", range(len(WIDE)))
@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("kw", [dict(), dict(causal=0, layout="head"), dict(n_layer=2, layer=1, pad_q=1, lse=False, extra_new=50, extra_len=99)])
def test_attention_of_many_f32_rows(K, pkg, shape, t, kw):
    """Enough rows for CTAs of 128 of them."""
    seqs, Hkv, g, D, ps = WIDE[shape]
    rows = max(n for n, _ in seqs) * g
    assert rows > 64 and -(-rows // 16) * Hkv * len(seqs) >= 6 * 148
    x = Attn(K, pkg, np.random.default_rng(60 + shape), seqs, Hkv, g, D, t, "f32", ps, **kw)
    pool = x.want_pool(x.c.view)
    x.run()
    x.check(pool)


def test_many_f32_rows_do_not_see_what_comes_later(K, pkg):
    """NaN and infinities in later tokens of the chunk reach only the queries from there on."""
    def make():
        return Attn(K, pkg, np.random.default_rng(2), [(200, 230)] * 4, 20, 1, 64, "f16", "f32", 16)
    x, y = make(), make()
    x.kn[100, 0], x.vn[100, 1, 3], x.vn[101, 2, 5] = float("nan"), float("inf"), float("nan")
    x.run()
    y.run()
    torch.cuda.synchronize()
    assert torch.equal(x.out[:100], y.out[:100]) and torch.equal(x.out[200:], y.out[200:]) and torch.equal(x.lse[:100], y.lse[:100])
    # (a weight is a sum of parts, the later ones of either sign or zero: its product with an infinite value is infinite or NaN)
    assert x.out[100:200, 0].isnan().all() and not x.out[100:200, 1, 3].isfinite().any() and x.out[101:200, 2, 5].isnan().all()
    rest = [i for i in range(64) if i != 5]
    assert torch.equal(x.out[100:200, 2][..., rest], y.out[100:200, 2][..., rest]) and torch.equal(x.out[100, 2], y.out[100, 2])
    assert torch.equal(x.out[:, 3:], y.out[:, 3:])


# The forms for many rows of 16-bit queries are taken where tiles are many (head_dim 64: 640 of 16 rows; 128: 512, or 250 000 tiles x keys)

@pytest.mark.parametrize("ps", [1, 3, 8, 16, 24, 48, 64, 128, 256, 512])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kw", [dict(t="f16"), dict(t="bf16", layout="head", causal=0), dict(t="bf16", scale=-0.3), dict(t="f16", scale=0.0, n_layer=2, layer=1, pad_q=1)])
def test_attention_of_many_16_bit_rows(K, pkg, ps, D, kw):
    t = kw["t"]
    x = Attn(K, pkg, np.random.default_rng(ps + D), [(150, 700), (1, 513), (90, 90), (256, 256), (0, 9), (100, 40)], 10, 1, D, t, t, ps, **{k: v for k, v in kw.items() if k != "t"})
    pool = x.want_pool(x.c.view)
    x.run()
    x.check(pool)


@pytest.mark.parametrize("seqs,Hkv,g,D,ps", [([(300, 2000), (129, 1300), (0, 0), (1, 900)], 2, 4, 128, 64), ([(70, 60003), (1, 3)], 1, 2, 128, 16), ([(64, 9000), (40, 7000)], 2, 1, 128, 24),
                                            ([(300, 4000), (129, 3300), (0, 0), (1, 5000)], 3, 1, 64, 16), ([(400, 2100)] * 3, 3, 3, 64, 100)])
def test_attention_of_many_16_bit_rows_split(K, pkg, seqs, Hkv, g, D, ps):
    """Few tiles over long contexts: split keys, and their join."""
    x = Attn(K, pkg, np.random.default_rng(len(seqs)), seqs, Hkv, g, D, "bf16", "bf16", ps)
    pool = x.want_pool(x.c.view)
    x.run()
    x.check(pool)


@pytest.mark.parametrize("ps", [64, 48])
def test_attention_of_many_16_bit_rows_and_pages_far_apart(K, pkg, far, ps):
    x = Attn(K, pkg, np.random.default_rng(ps), [(150, 260), (40, 300)], 2, 2, 128, "f16", "f16", ps, extra_len=9000)
    assert x.c.n_pages * x.c.pool.nb_page > 1 << 32
    pool = x.want_pool(x.c.view)
    x.run()
    x.check(pool)


@pytest.mark.parametrize("D", [64, 128])
def test_many_16_bit_rows_do_not_see_what_comes_later(K, pkg, D):
    def make():
        return Attn(K, pkg, np.random.default_rng(2), [(200, 230)] * 4, 20, 1, D, "f16", "f16", 16)
    x, y = make(), make()
    x.kn[100, 0], x.vn[100, 1, 3], x.vn[101, 2, 5] = float("nan"), float("inf"), float("nan")
    x.run()
    y.run()
    torch.cuda.synchronize()
    assert torch.equal(x.out[:100], y.out[:100]) and torch.equal(x.out[200:], y.out[200:]) and torch.equal(x.lse[:100], y.lse[:100])
    assert x.out[100:200, 0].isnan().all() and not x.out[100:200, 1, 3].isfinite().any() and x.out[101:200, 2, 5].isnan().all()
    rest = [i for i in range(D) if i != 5]
    assert torch.equal(x.out[100:200, 2][..., rest], y.out[100:200, 2][..., rest]) and torch.equal(x.out[100, 2], y.out[100, 2])
    assert torch.equal(x.out[:, 3:], y.out[:, 3:])


@pytest.mark.parametrize("D", [64, 128])
def test_many_16_bit_rows_with_huge_scores(K, pkg, D):
    """As test_attention_finite_but_huge_scores."""
    x = Attn(K, pkg, np.random.default_rng(D), [(130, 170)] * 5, 20, 1, D, "bf16", "bf16", 16, scale=1.0)
    x.q.mul_(2e17); x.kn.mul_(2e17)
    pool = x.want_pool(x.c.view)
    x.run()
    torch.cuda.synchronize()
    for i in (0, 4):
        k, v = (pool[j, 0].double().cpu().numpy()[x.tables[i, np.arange(170) // 16], np.arange(170) % 16] for j in (0, 1))
        out, _, _, _ = R.attention(x.q[130 * i:130 * (i + 1)].double().cpu().numpy(), k, v, 130, 170, 1.0, 1)
        assert np.all(np.abs(x.out[130 * i:130 * (i + 1)].double().cpu().numpy() - out) <= 2.0 ** -8 * np.abs(out) + 1e-30)


@pytest.mark.parametrize("D,heads", [(64, 20), (128, 10)])
def test_chunks_right_behind_what_makes_their_inputs(K, pkg, D, heads):
    """Queries, new rows, tables and lengths written by the launches just before, over and over, without a synchronisation between: attention
    begins while the store of its new rows still runs, but not before what came earlier."""
    rng = np.random.default_rng(D)
    seqs = [(200, 260), (130, 130), (90, 400), (256, 300)]
    xs = [Attn(K, pkg, rng, seqs, heads, 1, D, "f16", "f16", 16) for _ in range(2)]
    want = []
    for x in xs:
        x.run()
        torch.cuda.synchronize()
        want.append((x.out.clone(), x.lse.clone()))
    a = xs[0]
    sources = [(x.q.clone(), x.kn.clone(), x.vn.clone(), x.c.buf.clone(), x.dtab.clone(), x.dlen.clone()) for x in xs]
    got = []
    for i in range(12):
        for dst, src in zip((a.c.buf, a.kn, a.vn, a.dtab, a.dlen, a.q), (sources[i % 2][j] for j in (3, 1, 2, 4, 5, 0))):
            if dst.shape == src.shape:
                dst.copy_(src)
        if i % 3 == 0:
            a.out[:a.n_tok].zero_()
        a.run()
        got.append((a.out.clone(), a.lse.clone()))
    torch.cuda.synchronize()
    assert all(s[4].shape == a.dtab.shape and s[3].shape == a.c.buf.shape for s in sources)
    for i, g in enumerate(got):
        assert torch.equal(g[0], want[i % 2][0]) and torch.equal(g[1], want[i % 2][1]), i


@pytest.mark.parametrize("n_new,heads,qt", [(1, 2, "f16"), (3, 2, "f32"), (260, 20, "f16"), (260, 20, "f32")])
def test_attention_without_any_keys(K, pkg, n_new, heads, qt):
    """max_len 0, and lengths of 0 under a larger bound: zeros, lse -inf, nothing stored."""
    for max_len in (0, 500):
        x = Attn(K, pkg, np.random.default_rng(n_new), [(n_new, 300)] * 4, heads, 1, 64, "f16", qt, 16)
        before = x.c.view.clone()
        x.dlen.zero_()
        x.a.max_len = max_len
        n = K.b200_paged_attn_workspace(C.byref(x.c.pool), C.byref(x.a))
        x.ws = torch.zeros(max(n, 16), dtype=torch.uint8, device="cuda")
        x.a.workspace, x.a.workspace_bytes = p(x.ws), n
        x.run()
        torch.cuda.synchronize()
        assert torch.equal(torch.nan_to_num(x.c.view, 3.0), torch.nan_to_num(before, 3.0))
        assert (x.out[:x.n_tok] == 0).all() and (x.lse[:x.n_tok] == -np.inf).all() and (x.out[x.n_tok:] == 7).all()


def test_pages_of_no_rows(K, pkg):
    """No rows: update copies the counts, compact moves what other holders have."""
    c = Cache(pkg, np.random.default_rng(0), 20, 8)
    refs = np.zeros(20, int)
    refs[[3, 11, 17]] = 1, 2, 1
    before = c.view.clone()
    frm, f = c.state(pkg, np.zeros((0, 1), int), np.zeros(0, int), refs)
    to, t = c.state(pkg, np.zeros((0, 1), int), np.zeros(0, int), np.full(20, 99))
    status, remap = (torch.full((n,), 55, dtype=torch.int32, device="cuda") for n in (2, 20))
    n = K.b200_pages_workspace(0, 20)
    ws = torch.full((n,), 255, dtype=torch.uint8, device="cuda")
    assert K.b200_pages_update(C.byref(c.pool), C.byref(f), C.byref(t), None, None, None, p(status), p(ws), n, stream()) == 0
    torch.cuda.synchronize()
    assert status.tolist() == [0, 0] and np.array_equal(to["refs"].cpu().numpy(), refs) and torch.equal(c.view, before)
    assert K.b200_pages_compact(C.byref(c.pool), C.byref(f), C.byref(t), p(remap), p(status), p(ws), n, stream()) == 0
    torch.cuda.synchronize()
    got = remap.cpu().numpy()
    live = [int(i) for i in got[[3, 11, 17]]]
    assert status.tolist()[0] == 0 and sorted(live) == [0, 1, 2] and (got[refs == 0] == -1).all()
    for old, new in zip((3, 11, 17), live):
        assert torch.equal(c.view[:, :, new], before[:, :, old]) and int(to["refs"][new]) == refs[old]


def test_no_wait_ran_out(K, pkg):
    """After everything above (this process' launches so far)."""
    x = Attn(K, pkg, np.random.default_rng(0), [(300, 400)], 1, 1, 128, "f16", "f16", 16)
    x.run()
    torch.cuda.synchronize()
    assert K.b200_paged_attn_status() == 0
