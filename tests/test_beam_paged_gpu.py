"""Beam selection, state reordering, the paged cache and attention over it, through the C ABI, against plain 64-bit forms."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as R

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPE = {"f32": 0, "f16": 1, "bf16": 30}


@pytest.fixture(scope="module")
def K(pkg):
    assert torch.cuda.is_available(), "these tests need the B200; the kernel library has no CPU path"
    return pkg.kernels_lib()


def dev(a, dt=None):
    return torch.from_numpy(np.ascontiguousarray(a if dt is None else a.astype(dt))).cuda()


def p(t):
    return None if t is None else t.data_ptr()


def stream():
    return torch.cuda.current_stream().cuda_stream


# ---- selection ---------------------------------------------------------------------------------------------------

class Select:
    def __init__(self, K, pkg, logits, score, done, banned, eos, n_beam, offset=0, pad=0):
        """logits: torch [rows][V]; offset / pad: elements before the first row and between rows."""
        rows, V = logits.shape
        self.rows, self.K, self.n_beam = rows, K, n_beam
        flat = torch.full((offset + rows * (V + pad),), float("nan"), dtype=logits.dtype, device="cuda")
        view = flat[offset:].view(rows, V + pad)
        view[:, :V] = logits
        self.keep = [flat]
        self.score, self.done = dev(score, np.float32), None if done is None else dev(done, np.uint8)
        words = None
        if banned is not None:
            bits = np.zeros((banned.shape[0], -(-V // 32) * 32), bool)
            bits[:, :V] = banned
            words = dev(np.packbits(bits, axis=1, bitorder="little").view(np.int32))
        self.words = words
        self.o_score = torch.full((rows + 3,), 77.0, device="cuda")
        self.o_token, self.o_parent = (torch.full((rows + 3,), 77, dtype=torch.int32, device="cuda") for _ in range(2))
        self.o_done = torch.full((rows + 3,), 77, dtype=torch.uint8, device="cuda")
        n = K.b200_beam_select_workspace(rows // n_beam, n_beam, V)
        self.ws = torch.full((max(n, 16),), 255, dtype=torch.uint8, device="cuda")
        name = {v: k for k, v in DT.items()}[logits.dtype]
        self.a = pkg.BeamSelectArgs(logits=view.data_ptr(), type=TYPE[name], nb_row=(V + pad) * logits.element_size(), n_vocab=V, n_seq=rows // n_beam, n_beam=n_beam,
                                    score=p(self.score), done=p(self.done), eos=eos, banned=p(words), banned_stride=0 if words is None or words.shape[0] == 1 else words.shape[1],
                                    score_out=p(self.o_score), token_out=p(self.o_token), parent_out=p(self.o_parent), done_out=p(self.o_done),
                                    workspace=p(self.ws), workspace_bytes=n)

    def run(self):
        assert self.K.b200_beam_select(C.byref(self.a), stream()) == 0

    def got(self):
        torch.cuda.synchronize()
        assert (self.o_score[self.rows:] == 77).all() and (self.o_token[self.rows:] == 77).all() and (self.o_done[self.rows:] == 77).all()
        return {k: getattr(self, "o_" + k)[:self.rows].cpu().numpy() for k in ("score", "token", "parent", "done")}


def check_select(got, want):
    for k in ("token", "parent", "done"):
        assert np.array_equal(got[k], want[k]), k
    fin = np.isfinite(want["score"])
    assert np.array_equal(got["score"][~fin], want["score"][~fin])
    # each exponential is off by at most 2^-22 + |x| 2^-23 relative (argument scaled to base 2 in f32), |x| <= 40 where it counts: 5e-6
    # bounds the logarithm of the sum; the score is rounded once to f32
    assert np.all(np.abs(got["score"][fin] - want["score"][fin]) <= 5e-6 + np.abs(want["score"][fin]) * 2.0 ** -24)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n_seq,n_beam,V", [(1, 1, 1), (1, 5, 51866), (3, 4, 4096), (2, 32, 4097), (7, 3, 31), (2, 16, 9001), (1, 2, 70001), (40, 5, 777)])
def test_select(K, pkg, t, n_seq, n_beam, V):
    rng = np.random.default_rng(V + n_beam)
    x = torch.from_numpy(rng.standard_normal((n_seq * n_beam, V)) * 3).to(DT[t]).cuda()
    score = -rng.random(n_seq * n_beam) * 4 - 1
    score = score.astype(np.float32)
    done = (rng.random(n_seq * n_beam) < 0.3).astype(np.uint8)
    banned = rng.random((1, V)) < 0.2
    for d, m, off, pad in ((None, None, 0, 0), (done, banned, 1, 3), (done, rng.random((n_seq * n_beam, V)) < 0.5, 8, 1)):
        s = Select(K, pkg, x, score, d, m, min(5, V - 1), n_beam, off, pad)
        s.run()
        check_select(s.got(), R.beam_select(x.double().cpu().numpy(), score, d, m, min(5, V - 1), n_beam))


def test_select_where_candidates_are_special(K, pkg):
    """Slots not in use, rows of -inf and NaN, infinite logits, everything banned, ties inside a row and between equal rows of
    different alignment, an eos outside the vocabulary."""
    n_beam, V = 6, 5001                                   # an odd row length: every row has another alignment
    x = np.random.default_rng(0).standard_normal((5 * n_beam, V)).astype(np.float32)
    score = np.full(5 * n_beam, -1.5, np.float32)
    done = np.zeros(5 * n_beam, np.uint8)
    score[1:6] = -np.inf                                  # sequence 0: only its first beam is in use (the first step of a search)
    x[6:12] = x[6]                                        # sequence 1: six equal rows with equal scores
    x[6:12, 100:4600:450] = 9.0                           # ... and ties in every one of them
    x[12] = -np.inf; x[13] = np.nan; x[14, :] = -np.inf; x[14, 17] = 2.0      # sequence 2: few candidates
    score[15], done[16], score[17] = np.nan, 1, -np.inf
    x[18, 7] = np.inf; x[18, 9] = np.inf; x[19, 3] = np.nan; x[20, :] = 0.0; x[20, ::2] = -0.0   # sequence 3
    done[24:30] = 1                                       # sequence 4: all done
    banned = np.zeros((5 * n_beam, V), bool)
    banned[21] = True
    for eos in (3, -1, V + 5):
        s = Select(K, pkg, torch.from_numpy(x).cuda(), score, done, banned, eos, n_beam)
        s.run()
        with np.errstate(all="ignore"):
            check_select(s.got(), R.beam_select(x, score, done, banned, eos, n_beam))


def test_select_in_place_on_a_stream_and_captured(K, pkg):
    """score / done updated in place, on another stream than the default, replayed from a graph with new inputs."""
    rng = np.random.default_rng(5)
    x = torch.from_numpy(rng.standard_normal((10, 6000)).astype(np.float32)).cuda()
    s = Select(K, pkg, x, -rng.random(10), np.zeros(10), None, 7, 5)
    s.a.score_out, s.a.done_out = s.a.score, s.a.done
    first_score, first_done = s.score.clone(), s.done.clone()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        s.run()
        s.score.copy_(first_score); s.done.copy_(first_done)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            s.run()
        for seed in (1, 2):
            x2 = torch.from_numpy(np.random.default_rng(seed).standard_normal((10, 6000)).astype(np.float32)).cuda()
            s.keep[0].view(10, 6000).copy_(x2)
            before, d0 = s.score.cpu().numpy(), s.done.cpu().numpy()
            g.replay()
            st.synchronize()
            want = R.beam_select(x2.cpu().numpy(), before, d0, None, 7, 5)
            got = dict(score=s.score.cpu().numpy(), token=s.o_token[:10].cpu().numpy(), parent=s.o_parent[:10].cpu().numpy(), done=s.done.cpu().numpy())
            check_select(got, want)


# ---- reordering --------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("n_seq,n_beam,outer,row,used,off", [(1, 5, 3, 512, 512, 0), (4, 2, 1, 48, 47, 0), (2, 8, 2, 100, 97, 4), (3, 16, 5, 33, 33, 1),
                                                            (2, 32, 2, 4096, 4000, 16), (5, 1, 2, 64, 64, 0), (2, 3, 4, 20000, 19999, 0)])
def test_reorder(K, pkg, n_seq, n_beam, outer, row, used, off):
    rng = np.random.default_rng(row + n_beam)
    rows = n_seq * n_beam
    parent = rng.integers(-1, n_beam + 1, rows).astype(np.int32)          # -1 and n_beam: left as they are
    data = rng.integers(0, 256, off + outer * rows * row, dtype=np.uint8)
    hist = rng.integers(0, 50000, (rows, 9), dtype=np.int32)
    d, h = dev(data), dev(hist)
    blocks = (pkg.BeamBlock * 2)(pkg.BeamBlock(base=d.data_ptr() + off, n_outer=outer, nb_outer=rows * row, nb_row=row, row_bytes=used),
                                 pkg.BeamBlock(base=h.data_ptr(), n_outer=1, nb_outer=0, nb_row=36, row_bytes=28))
    assert K.b200_beam_reorder(blocks, 2, dev(parent).data_ptr(), n_seq, n_beam, stream()) == 0
    torch.cuda.synchronize()
    src = np.arange(rows)
    ok = (parent >= 0) & (parent < n_beam)
    src[ok] = src[ok] // n_beam * n_beam + parent[ok]
    want = data.copy()
    v, o = want[off:].reshape(outer, rows, row), data[off:].reshape(outer, rows, row)
    v[:, :, :used] = o[:, src, :used]
    assert np.array_equal(d.cpu().numpy(), want)
    wh = hist.copy()
    wh[:, :7] = hist[src, :7]
    assert np.array_equal(h.cpu().numpy(), wh)


def test_reorder_with_layers_inside_a_row(K, pkg):
    """[row][layer][bytes]: the outer index runs inside a row."""
    rng = np.random.default_rng(3)
    data = rng.integers(0, 256, (6, 4, 80), dtype=np.uint8)
    d, parent = dev(data), np.array([2, 0, 0, 1, 1, 2], np.int32)
    b = (pkg.BeamBlock * 1)(pkg.BeamBlock(base=p(d), n_outer=4, nb_outer=80, nb_row=320, row_bytes=64))
    assert K.b200_beam_reorder(b, 1, dev(parent).data_ptr(), 2, 3, stream()) == 0
    want = data.copy()
    want[:, :, :64] = data[[2, 0, 0, 4, 4, 5], :, :64]
    assert np.array_equal(d.cpu().numpy(), want)


# ---- pages -------------------------------------------------------------------------------------------------------

class Cache:
    """A pool of random values and a random state of rows over it; `layout` token- or head-major pages with gaps between them."""

    def __init__(self, pkg, rng, n_pages, ps, Hkv=2, D=64, t="f16", n_layer=1, layout="tok", gap=0):
        self.n_pages, self.ps, self.Hkv, self.D, self.t, self.n_layer = n_pages, ps, Hkv, D, t, n_layer
        shape = (ps, Hkv) if layout == "tok" else (Hkv, ps)
        page = ps * Hkv * D + gap * 8
        self.buf = torch.from_numpy(rng.standard_normal((2, n_layer, n_pages, page))).to(DT[t]).cuda()
        self.view = self.buf[..., : ps * Hkv * D].unflatten(-1, (*shape, D))
        if layout != "tok":
            self.view = self.view.transpose(3, 4)          # [2][layer][page][tok][head][D] either way
        es = 2
        self.pool = pkg.PagePool(k=self.buf[0].data_ptr(), v=self.buf[1].data_ptr(), type=TYPE[t], n_layer=n_layer, n_pages=n_pages, page_size=ps, n_head_kv=Hkv, head_dim=D,
                                 nb_layer=n_pages * page * es, nb_page=page * es, nb_tok=(Hkv * D if layout == "tok" else D) * es,
                                 nb_head=(D if layout == "tok" else ps * D) * es)

    def state(self, pkg, tables, lens, refs):
        t = dict(tables=dev(tables, np.int32), lens=dev(lens, np.int32), refs=dev(refs, np.int32))
        return t, pkg.PageState(tables=p(t["tables"]), lens=p(t["lens"]), refs=p(t["refs"]), n_rows=len(lens), table_stride=tables.shape[1])


def random_state(rng, n_groups, beams, ps, max_len, n_pages, width, extra=False):
    """Groups of rows with common first pages."""
    ids = list(rng.permutation(n_pages))
    rows = n_groups * beams
    tables, lens = np.full((rows, width), -1), np.zeros(rows, int)
    for g in range(n_groups):
        n = int(rng.integers(0, max_len + 1))
        common = [ids.pop() for _ in range(int(rng.integers(0, R.ceil(n, ps) + 1)))]
        for b in range(beams):
            r = g * beams + b
            mine = common + [ids.pop() for _ in range(R.ceil(n, ps) - len(common))]
            tables[r, :len(mine)] = mine
            lens[r] = n
    refs = np.bincount(tables[tables >= 0].astype(int), minlength=n_pages)
    if extra:
        refs[tables[0, 0] if lens[0] else 0] += 1           # a holder that the tables do not show
    return tables, lens, refs


def run_update(K, pkg, c, tables, lens, refs, parent, keep, new, pool=None, data=True):
    frm, f = c.state(pkg, tables, lens, refs)
    to, t = c.state(pkg, np.full_like(tables, 99), np.full_like(lens, 99), np.full_like(refs, 99))
    status = torch.full((2,), 55, dtype=torch.int32, device="cuda")
    n = K.b200_pages_workspace(len(lens), c.n_pages)
    ws = torch.full((n,), 255, dtype=torch.uint8, device="cuda")
    arg = [None if a is None else dev(np.asarray(a), np.int32) for a in (parent, keep, new)]
    assert K.b200_pages_update(C.byref(pool or c.pool), C.byref(f), C.byref(t), *(p(a) for a in arg), p(status), p(ws), n, stream()) == 0
    torch.cuda.synchronize()
    for k, a in (("tables", tables), ("lens", lens), ("refs", refs)):
        assert np.array_equal(frm[k].cpu().numpy(), a), "from was written"
    return {k: v.cpu().numpy() for k, v in to.items()}, status.tolist(), (ws, n)


def check_update(c, before, got, status, want):
    tables, lens, refs, copies, st = want
    assert status == [st, len(copies)]
    assert np.array_equal(got["tables"], tables) and np.array_equal(got["lens"], lens) and np.array_equal(got["refs"], refs)
    after = before.clone()
    for s, d, n in copies:
        after[:, :, d, :n] = before[:, :, s, :n]
    assert torch.equal(c.view, after)


@pytest.mark.parametrize("n_groups,beams,ps,max_len,width,layout", [(1, 5, 16, 60, 6, "tok"), (3, 4, 7, 40, 9, "head"), (1, 1, 1, 3, 5, "tok"), (40, 5, 8, 200, 30, "tok"),
                                                                   (1, 2, 64, 63, 2, "head"), (400, 3, 4, 90, 30, "tok"), (2, 8, 16, 0, 3, "tok")])
def test_update(K, pkg, n_groups, beams, ps, max_len, width, layout):
    for seed in range(3):
        rng = np.random.default_rng(seed * 1000 + n_groups)
        rows = n_groups * beams
        n_pages = rows * (R.ceil(max_len, ps) + 2) + 3
        c = Cache(pkg, rng, n_pages, ps, layout=layout, n_layer=2, gap=1, D=128 if seed == 1 else 64, t="bf16" if seed == 2 else "f16")
        tables, lens, refs = random_state(rng, n_groups, beams, ps, max_len, n_pages, width, extra=seed == 2)
        parent = np.arange(rows) // beams * beams + rng.integers(0, beams, rows)
        keep, new = lens[parent].copy(), np.ones(rows, int)
        if seed:
            cut = rng.random(rows) < 0.4
            keep[cut] = (keep[cut] * rng.random(cut.sum())).astype(int)
            new[rng.random(rows) < 0.3] = 0
            many = rng.random(rows) < 0.2
            new[many] = rng.integers(0, width * ps + 1 - keep.max(), many.sum())
            gone = rng.random(rows) < 0.1
            keep[gone] = new[gone] = 0
        before = c.view.clone()
        got, status, _ = run_update(K, pkg, c, tables, lens, refs, parent, keep, new)
        want = R.pages_update(tables, lens, refs, parent, keep, new, ps)
        check_update(c, before, got, status, want)


def test_update_refuses_on_the_device(K, pkg):
    """Requests that cannot be met leave a copy of the state and say why."""
    rng = np.random.default_rng(1)
    c = Cache(pkg, rng, 12, 4)
    tables = np.array([[3, 5, -1, -1], [3, 7, 9, -1]])
    lens, refs = np.array([8, 10]), np.bincount([3, 5, 3, 7, 9], minlength=12)
    before = c.view.clone()
    for parent, keep, new in (([0, 2], [8, 0], [0, 0]), ([0, -1], [8, 0], [0, 0]), ([0, 0], [8, 9], [0, 0]), ([0, 1], [-1, 0], [0, 0]), ([0, 1], [8, 8], [0, -2]),
                              ([0, 1], [8, 8], [9, 0]), ([1, 1], [8, 8], [2**31 - 1, 0])):
        got, status, _ = run_update(K, pkg, c, tables, lens, refs, parent, keep, new)
        check_update(c, before, got, status, (tables, lens, refs, [], -1))
    bad = tables.copy()
    bad[1, 1] = 12
    got, status, _ = run_update(K, pkg, c, bad, lens, refs, None, [8, 8], [0, 0])
    check_update(c, before, got, status, (bad, lens, refs, [], -1))
    full = np.ones(12, int)
    full[[0, 1]] = 0                                       # two free pages, three wanted
    got, status, _ = run_update(K, pkg, c, tables, lens, full, None, [8, 10], [5, 3])
    check_update(c, before, got, status, (tables, lens, full, [], 1))


def test_update_without_parents_tables_only_and_copies_elsewhere(K, pkg):
    rng = np.random.default_rng(9)
    c, other = Cache(pkg, rng, 30, 8), Cache(pkg, rng, 30, 8, Hkv=3, D=128, t="bf16", n_layer=3)
    tables, lens, refs = np.array([[1, 2, -1, -1], [1, 2, -1, -1], [1, 4, 6, -1]]), np.array([13, 13, 20]), np.zeros(30, int)
    refs[[1, 2, 4, 6]] = 3, 2, 1, 1
    want = R.pages_update(tables, lens, refs, [0, 1, 2], lens, [1, 2, 3], 8)
    before, ob = c.view.clone(), other.view.clone()
    no_data = type(c.pool).from_buffer_copy(c.pool)
    no_data.k = no_data.v = None
    got, status, (ws, n) = run_update(K, pkg, c, tables, lens, refs, None, lens, [1, 2, 3], pool=no_data)
    assert torch.equal(c.view, before) and status == [0, 1] and np.array_equal(got["tables"], want[0]) and np.array_equal(got["refs"], want[2])
    assert K.b200_pages_copy(C.byref(other.pool), 3, p(ws), n, stream()) == 0
    assert K.b200_pages_copy(C.byref(c.pool), 3, p(ws), n, stream()) == 0
    torch.cuda.synchronize()
    check_update(c, before, got, status, want)
    check_update(other, ob, got, status, want)


@pytest.mark.parametrize("n_groups,beams,ps,max_len,n_pages", [(1, 1, 4, 9, 8), (6, 2, 16, 100, 200), (200, 3, 8, 60, 9000), (3, 1, 5, 0, 6)])
@pytest.mark.parametrize("layout", ["tok", "head"])
def test_compact(K, pkg, n_groups, beams, ps, max_len, n_pages, layout):
    rng = np.random.default_rng(n_pages)
    width = R.ceil(max_len, ps) + 1
    c = Cache(pkg, rng, n_pages, ps, layout=layout, n_layer=2)
    tables, lens, refs = random_state(rng, n_groups, beams, ps, max_len, n_pages, width, extra=max_len > 0)
    frm, f = c.state(pkg, tables, lens, refs)
    to, t = c.state(pkg, np.full_like(tables, 99), np.full_like(lens, 99), np.full_like(refs, 99))
    status, remap = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    n = K.b200_pages_workspace(len(lens), n_pages)
    ws = torch.full((n,), 255, dtype=torch.uint8, device="cuda")
    before = c.view.clone()
    assert K.b200_pages_compact(C.byref(c.pool), C.byref(f), C.byref(t), p(remap), p(status), p(ws), n, stream()) == 0
    torch.cuda.synchronize()
    wt, wl, wr, wm, moves = R.pages_compact(tables, lens, refs, ps)
    assert status.tolist() == [0, len(moves)] and np.array_equal(remap.cpu().numpy(), wm)
    assert np.array_equal(to["tables"].cpu().numpy(), wt) and np.array_equal(to["lens"].cpu().numpy(), wl) and np.array_equal(to["refs"].cpu().numpy(), wr)
    for a, b in moves:
        assert torch.equal(c.view[:, :, b], before[:, :, a])
    rest = [i for i in range(n_pages) if i not in {b for _, b in moves}]
    assert torch.equal(c.view[:, :, rest], before[:, :, rest])
    if max_len:                                            # a table that names a free page is refused
        bad = tables.copy()
        row = int(np.argmax(lens))
        bad[row, 0] = int(np.argmin(refs))
        frm, f = c.state(pkg, bad, lens, refs)
        assert K.b200_pages_compact(C.byref(c.pool), C.byref(f), C.byref(t), p(remap), p(status), p(ws), n, stream()) == 0
        torch.cuda.synchronize()
        assert status.tolist() == [-1, 0] and np.array_equal(to["tables"].cpu().numpy(), bad) and np.array_equal(to["refs"].cpu().numpy(), refs)
        assert np.array_equal(remap.cpu().numpy(), np.where(refs != 0, np.arange(n_pages), -1))


# ---- attention ---------------------------------------------------------------------------------------------------

class Attn:
    def __init__(self, K, pkg, rng, seqs, Hkv, g, D, t, qt, ps, layout="tok", causal=1, scale=None, store=True, lse=True, extra_len=0, extra_new=0, n_layer=1, layer=0, pad_q=0):
        """seqs: [(n_new, length)]; extra_*: how far the host's bounds lie above the true ones."""
        self.K, self.pkg, self.seqs, self.causal, self.t, self.qt, self.layer = K, pkg, seqs, causal, t, qt, layer
        H = Hkv * g
        self.scale = 1 / np.sqrt(D) if scale is None else scale
        need = [R.ceil(n, ps) for _, n in seqs]
        self.c = Cache(pkg, rng, sum(need) + 2, ps, Hkv, D, t, n_layer=n_layer, layout=layout, gap=2)
        ids = rng.permutation(self.c.n_pages)
        self.tables = np.full((len(seqs), max(need) + 1), -1, np.int32)
        at = 0
        for i, n in enumerate(need):
            self.tables[i, :n] = ids[at:at + n]
            at += n
        # pages behind a sequence's end hold what no query may see
        bad = torch.tensor([float("nan"), float("inf")], device="cuda", dtype=DT[t])
        for i, (_, n) in enumerate(seqs):
            if n % ps:
                self.c.view[:, :, int(self.tables[i, n // ps]), n % ps:] = bad.repeat(D // 2)
        for i in ids[at:]:
            self.c.view[:, :, int(i)] = float("nan")
        n_tok = sum(n for n, _ in seqs)
        self.start = np.concatenate([[0], np.cumsum([n for n, _ in seqs])]).astype(np.int32)
        mk = lambda h, pad: torch.from_numpy(rng.standard_normal((max(n_tok, 1), h + pad, D))).to(DT[qt]).cuda()  # noqa: E731
        self.q, self.kn, self.vn = mk(H, pad_q), mk(Hkv, 0), mk(Hkv, 0)
        self.out = torch.full((n_tok + 2, H, D), 7.0, dtype=DT[qt], device="cuda")
        self.lse = torch.full((n_tok + 2, H), 7.0, device="cuda") if lse else None
        es = self.q.element_size()
        self.dtab, self.dlen, self.dstart = dev(self.tables), dev(np.array([n for _, n in seqs], np.int32)), dev(self.start)
        self.a = pkg.PagedAttnArgs(q=p(self.q), q_type=TYPE[qt], nb_q_tok=(H + pad_q) * D * es, nb_q_head=D * es, dst=p(self.out), nb_dst_tok=H * D * es, nb_dst_head=D * es,
                                   k_new=p(self.kn) if store else None, v_new=p(self.vn) if store else None, nb_new_tok=Hkv * D * es, nb_new_head=D * es, layer=layer,
                                   tables=p(self.dtab), table_stride=self.tables.shape[1], lens=p(self.dlen), q_start=p(self.dstart), n_tok=n_tok, n_seq=len(seqs),
                                   n_head=H, max_new=max(n for n, _ in seqs) + extra_new, max_len=max(n for _, n in seqs) + extra_len, causal=causal, scale=self.scale,
                                   lse=p(self.lse))
        n = K.b200_paged_attn_workspace(C.byref(self.c.pool), C.byref(self.a))
        self.ws = torch.full((max(n, 16),), 255, dtype=torch.uint8, device="cuda")
        self.a.workspace, self.a.workspace_bytes = p(self.ws), n
        self.store, self.n_tok, self.H, self.Hkv, self.D, self.ps = store, n_tok, H, Hkv, D, ps

    def run(self):
        assert self.K.b200_paged_attn(C.byref(self.c.pool), C.byref(self.a), stream()) == 0

    def want_pool(self, before):
        w = before.clone()
        if self.store:
            for i, (n_new, n) in enumerate(self.seqs):
                for t in range(n_new):
                    pos = n - n_new + t
                    if pos >= 0:
                        for j, x in enumerate((self.kn, self.vn)):
                            w[j, self.layer, int(self.tables[i, pos // self.ps]), pos % self.ps] = x[int(self.start[i]) + t].to(w.dtype)
        return w

    def check(self, pool):
        torch.cuda.synchronize()
        assert torch.equal(torch.nan_to_num(self.c.view, 3.0), torch.nan_to_num(pool, 3.0)), "the pages do not hold what was stored, or more"
        assert (self.out[self.n_tok:] == 7).all(), "rows behind the last token were written"
        u = torch.finfo(DT[self.qt]).eps / 2
        up = torch.finfo(DT[self.t]).eps / 2 if self.qt != "f32" else 0.0
        vals = pool[:, self.layer].double().cpu().numpy()
        for i, (n_new, n) in enumerate(self.seqs):
            if n_new == 0:
                continue
            pg = self.tables[i, np.arange(n) // self.ps]
            k, v = (vals[j][pg, np.arange(n) % self.ps] if n else np.zeros((0, self.Hkv, self.D)) for j in (0, 1))
            sl = slice(int(self.start[i]), int(self.start[i]) + n_new)
            out, lse, mag, reach = R.attention(self.q[sl, :self.H].double().cpu().numpy(), k, v, n_new, n, self.scale, self.causal)
            got = self.out[sl].double().cpu().numpy()
            # a score is a sum of D products in f32, scaled: off by (D + 4) 2^-24 times the sum of their magnitudes (reach); a weight is
            # off by that times 2 (numerator and sum), its exponential by 2^-22, and by `up` where it is rounded to the pool's type;
            # sums over n keys and over the parts that are joined add (n + 80) 2^-24; the result is rounded once
            w = 2 * (self.D + 4) * 2.0 ** -24 * reach + 2.0 ** -21 + (n + 80) * 2.0 ** -23
            tol = u * np.abs(out) + (w[..., None] + up * (1 + u)) * mag + 1e-30
            if self.qt == "f16":
                tol += 2.0 ** -25                          # f16 subnormals
            bad = ~(np.abs(got - out) <= tol)
            assert not bad.any(), f"sequence {i}: {bad.sum()} of {bad.size} off, by {np.abs(got - out)[bad].max():.3g}, first at {np.argwhere(bad)[0]}"
            if self.lse is not None:
                gl = self.lse[sl].double().cpu().numpy()
                fin = np.isfinite(lse)
                assert np.array_equal(gl[~fin], lse[~fin])
                assert np.all(np.abs(gl[fin] - lse[fin]) <= w[fin] + 2.0 ** -21 * (1 + np.abs(lse[fin])))


SHAPES = [
    # seqs, Hkv, g, D, ps
    ([(1, 1)], 1, 1, 64, 16),
    ([(1, 448)] * 5, 20, 1, 64, 16),
    ([(1, 37), (1, 5), (0, 0), (1, 300), (1, 0)], 2, 4, 128, 16),
    ([(3, 3), (1, 130), (2, 65)], 3, 5, 64, 5),
    ([(17, 17), (40, 200), (1, 1), (5, 4)], 2, 3, 64, 8),
    ([(130, 130), (224, 224), (7, 500)], 4, 1, 64, 16),
    ([(300, 700), (129, 129)], 2, 4, 128, 64),
    ([(1, 3000), (2, 1999)], 1, 8, 128, 100),
    ([(64, 1025)], 1, 16, 128, 1),
    ([(260, 515), (0, 40), (33, 33)], 1, 2, 128, 128),
    ([(16, 100), (9, 9), (2, 300), (0, 7), (16, 17)], 2, 4, 64, 16),
    ([(1, 5000), (1, 1), (0, 0), (1, 777), (1, 4096), (1, 64)], 3, 2, 128, 16),
    ([(4, 3001), (1, 3), (3, 2500)], 2, 7, 64, 24),
    ([(300, 2000), (129, 1300), (0, 0), (1, 900)], 2, 4, 128, 64),
    ([(200, 1500), (70, 700), (5, 9), (3, 2)], 3, 3, 64, 16),
    ([(150, 1200), (0, 0), (40, 2100)], 2, 2, 128, 24),
    ([(300, 1100), (280, 1030), (0, 0), (290, 1200), (257, 1025)], 20, 2, 128, 32),
    ([(260, 520)] * 3 + [(500, 700), (0, 3), (390, 1000)] + [(257, 514)] * 6, 20, 1, 64, 16),
]


@pytest.mark.parametrize("shape", range(len(SHAPES)))
@pytest.mark.parametrize("t,qt", [("f16", "f16"), ("bf16", "bf16"), ("f16", "f32"), ("bf16", "f32")])
def test_attention(K, pkg, shape, t, qt):
    seqs, Hkv, g, D, ps = SHAPES[shape]
    x = Attn(K, pkg, np.random.default_rng(shape), seqs, Hkv, g, D, t, qt, ps)
    pool = x.want_pool(x.c.view)
    x.run()
    x.check(pool)


@pytest.mark.parametrize("qt", ["f16", "f32"])
@pytest.mark.parametrize("kw", [dict(causal=0), dict(layout="head"), dict(store=False, lse=False), dict(extra_len=2000, extra_new=70), dict(n_layer=3, layer=2, pad_q=3),
                                dict(scale=-0.5), dict(scale=0.0)])
@pytest.mark.parametrize("shape", [2, 4, 6])
def test_attention_forms(K, pkg, qt, kw, shape):
    seqs, Hkv, g, D, ps = SHAPES[shape]
    x = Attn(K, pkg, np.random.default_rng(50 + shape), seqs, Hkv, g, D, "f16", qt, ps, **kw)
    pool = x.want_pool(x.c.view)
    if not x.store:                                        # the pages hold the new tokens already
        pool = x.c.view.clone()
    x.run()
    x.check(pool)


@pytest.mark.parametrize("qt", ["bf16", "f32"])
@pytest.mark.parametrize("n_new", [4, 200])
def test_what_a_query_does_not_see_has_no_effect(K, pkg, qt, n_new):
    """NaN and infinities in later tokens of the same chunk reach only the queries from there on."""
    x = Attn(K, pkg, np.random.default_rng(7), [(n_new, n_new + 9)], 2, 2, 64, "bf16", qt, 16)
    bad = n_new // 2
    x.kn[bad, 0], x.vn[bad, 0, 3], x.vn[bad + 1, 1, 5] = float("nan"), float("inf"), float("nan")
    x.run()
    got = x.out.double().cpu().numpy()
    y = Attn(K, pkg, np.random.default_rng(7), [(n_new, n_new + 9)], 2, 2, 64, "bf16", qt, 16)
    y.run()
    torch.cuda.synchronize()
    assert torch.equal(x.out[:bad], y.out[:bad]) and torch.equal(x.lse[:bad], y.lse[:bad])
    assert np.isnan(got[bad:n_new, 0:2]).all()             # the heads that read the NaN key
    assert torch.equal(x.out[bad, 2:], y.out[bad, 2:])     # the other head's values are clean up to here
    assert np.isnan(got[bad + 1:n_new, 2:, 5]).all()
    rest = [i for i in range(64) if i != 5]
    assert torch.equal(x.out[bad + 1:n_new, 2:][..., rest], y.out[bad + 1:n_new, 2:][..., rest])


def test_attention_same_bits_every_time_on_streams_and_in_graphs(K, pkg):
    """Two captured graphs that share a workspace, replayed in turn on a side stream, give the bits of plain calls."""
    for seqs in ([(1, 2000)] * 3, [(200, 900), (64, 64)]):
        xs = [Attn(K, pkg, np.random.default_rng(s), seqs, 2, 4, 128, "bf16", "bf16", 16) for s in (1, 2)]
        xs[1].ws, xs[1].a.workspace = xs[0].ws, xs[0].a.workspace
        want = []
        for x in xs:
            x.run()
            torch.cuda.synchronize()
            want.append((x.out.clone(), x.lse.clone()))
        st, graphs = torch.cuda.Stream(), []
        with torch.cuda.stream(st):
            for x in xs:
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=st):
                    x.run()
                graphs.append(g)
            for x in xs:
                x.out[:x.n_tok].zero_(); x.lse[:x.n_tok].zero_()
            for _ in range(3):
                for g in graphs:
                    g.replay()
            st.synchronize()
        for x, (o, l) in zip(xs, want):
            assert torch.equal(x.out, o) and torch.equal(x.lse, l)


def test_attention_bad_pages_and_lengths(K, pkg):
    """Table entries outside the pool read as zeros and store nothing; lengths beyond the tables are cut off."""
    x = Attn(K, pkg, np.random.default_rng(3), [(2, 40), (1, 20)], 2, 2, 64, "f16", "f16", 16)
    t = x.tables.copy()
    t[0, 0], t[0, 2] = x.c.n_pages + 5, -7                 # a page of the past, and the page of the new tokens
    x.dtab.copy_(torch.from_numpy(t))
    before = x.c.view.clone()
    x.run()
    torch.cuda.synchronize()
    pool = before.clone()
    pool[0, 0, int(t[1, 1]), 3], pool[1, 0, int(t[1, 1]), 3] = x.kn[2], x.vn[2]
    assert torch.equal(torch.nan_to_num(x.c.view, 3.0), torch.nan_to_num(pool, 3.0))
    k = np.zeros((2, 40, 2, 64))
    k[:, 16:32] = pool[:, 0, int(t[0, 1])].double().cpu().numpy()
    out, _, mag, _ = R.attention(x.q[:2].double().cpu().numpy(), k[0], k[1], 2, 40, x.scale, 1)
    assert np.all(np.abs(x.out[:2].double().cpu().numpy() - out) <= 2.0 ** -11 * np.abs(out) + (2.0 ** -11 + 1e-4) * mag + 2.0 ** -25)
    x.dlen.fill_(1000)                                     # beyond table_stride * page_size and beyond max_len
    x.run()
    torch.cuda.synchronize()


# ---- together ----------------------------------------------------------------------------------------------------

def test_a_beam_search_step_by_step(K, pkg):
    """Prompt, then beam steps: attention over the pages -> logits -> selection -> pages fork and grow, histories follow; every step's
    attention is checked against dense caches kept per beam on the host, the tables and counts against the plain form; at the end the pool is
    compacted and one more step gives what it gave before."""
    rng = np.random.default_rng(11)
    n_seq, B, Hkv, g, D, ps, V, width = 2, 3, 2, 2, 64, 4, 500, 12
    rows, H = n_seq * B, Hkv * g
    c = Cache(pkg, rng, 60, ps, Hkv, D, "f16")
    lens = np.zeros(rows, np.int32)
    tables, refs = np.full((rows, width), -1, np.int32), np.zeros(60, np.int32)
    frm, f = c.state(pkg, tables, lens, refs)
    to, t = c.state(pkg, tables, lens, refs)
    status = torch.zeros(2, dtype=torch.int32, device="cuda")
    n_ws = K.b200_pages_workspace(rows, 60)
    ws = torch.empty(n_ws, dtype=torch.uint8, device="cuda")
    dense = [[np.zeros((0, Hkv, D)), np.zeros((0, Hkv, D))] for _ in range(rows)]
    hist = torch.zeros(rows, 16, dtype=torch.int32, device="cuda")
    score = torch.tensor([0.0, -np.inf, -np.inf] * n_seq, device="cuda")
    done = torch.zeros(rows, dtype=torch.uint8, device="cuda")
    token, parent = (torch.zeros(rows, dtype=torch.int32, device="cuda") for _ in range(2))
    W = torch.from_numpy(rng.standard_normal((H * D, V))).float().cuda()
    sel_n = K.b200_beam_select_workspace(n_seq, B, V)
    sel_ws = torch.empty(sel_n, dtype=torch.uint8, device="cuda")
    step_new = [np.array([5, 0, 0, 7, 0, 0])] + [np.ones(rows, int)] * 6
    par = np.arange(rows)
    for step, new in enumerate(step_new):
        keep = lens[par]
        want = R.pages_update(tables, lens, refs, par, keep, new, ps)
        arg = [dev(a, np.int32) for a in (par, keep, new)]
        assert K.b200_pages_update(C.byref(c.pool), C.byref(f), C.byref(t), *(p(a) for a in arg), p(status), p(ws), n_ws, stream()) == 0
        frm, f, to, t = to, t, frm, f
        tables, lens, refs = (want[i].astype(np.int32) for i in range(3))
        assert status.tolist() == [0, len(want[3])]
        for k, w in (("tables", tables), ("lens", lens), ("refs", refs)):
            assert np.array_equal(frm[k].cpu().numpy(), w)
        n_tok = int(new.sum())
        start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        q, kn, vn = (torch.from_numpy(rng.standard_normal((n_tok, h, D))).half().cuda() for h in (H, Hkv, Hkv))
        out = torch.empty(n_tok, H, D, dtype=torch.float16, device="cuda")
        ds = dev(start)
        a = pkg.PagedAttnArgs(q=p(q), q_type=1, nb_q_tok=H * D * 2, nb_q_head=D * 2, dst=p(out), nb_dst_tok=H * D * 2, nb_dst_head=D * 2, k_new=p(kn), v_new=p(vn),
                              nb_new_tok=Hkv * D * 2, nb_new_head=D * 2, layer=0, tables=p(frm["tables"]), table_stride=width, lens=p(frm["lens"]), q_start=p(ds), n_tok=n_tok,
                              n_seq=rows, n_head=H, max_new=int(new.max()), max_len=int(lens.max()), causal=1, scale=0.125)
        n = K.b200_paged_attn_workspace(C.byref(c.pool), C.byref(a))
        aws = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
        a.workspace, a.workspace_bytes = p(aws), n
        assert K.b200_paged_attn(C.byref(c.pool), C.byref(a), stream()) == 0
        dense = [[np.concatenate([dense[par[r]][j], x[start[r]:start[r + 1]].double().cpu().numpy()]) for j, x in enumerate((kn, vn))] for r in range(rows)]
        got = out.double().cpu().numpy()
        for r in range(rows):
            sl = slice(start[r], start[r + 1])
            o, _, mag, _ = R.attention(q[sl].double().cpu().numpy(), *dense[r], int(new[r]), len(dense[r][0]), 0.125, 1)
            assert np.all(np.abs(got[sl] - o) <= 2.0 ** -11 * np.abs(o) + (2.0 ** -11 + 1e-4) * mag + 2.0 ** -25), (step, r)
        last = torch.zeros(rows, H * D, device="cuda")
        has = np.flatnonzero(new)
        last[torch.from_numpy(has).cuda()] = out[torch.from_numpy(start[1:][has].astype(np.int64) - 1).cuda()].view(len(has), -1).float()
        logits = (last @ W).contiguous()
        before, d0 = score.cpu().numpy(), done.cpu().numpy()
        s = pkg.BeamSelectArgs(logits=p(logits), type=0, nb_row=V * 4, n_vocab=V, n_seq=n_seq, n_beam=B, score=p(score), done=p(done), eos=3, score_out=p(score), token_out=p(token),
                               parent_out=p(parent), done_out=p(done), workspace=p(sel_ws), workspace_bytes=sel_n)
        assert K.b200_beam_select(C.byref(s), stream()) == 0
        check_select(dict(score=score.cpu().numpy(), token=token.cpu().numpy(), parent=parent.cpu().numpy(), done=done.cpu().numpy()),
                     R.beam_select(logits.double().cpu().numpy(), before, d0, None, 3, B))
        hb = hist.cpu().numpy()
        blk = (pkg.BeamBlock * 1)(pkg.BeamBlock(base=p(hist), n_outer=1, nb_outer=0, nb_row=64, row_bytes=64))
        assert K.b200_beam_reorder(blk, 1, p(parent), n_seq, B, stream()) == 0
        par = np.arange(rows) // B * B + np.maximum(parent.cpu().numpy(), 0)
        assert np.array_equal(hist.cpu().numpy(), hb[par])
        hist[:, step] = token
    remap = torch.empty(60, dtype=torch.int32, device="cuda")
    assert K.b200_pages_compact(C.byref(c.pool), C.byref(f), C.byref(t), p(remap), p(status), p(ws), n_ws, stream()) == 0
    again = torch.empty_like(out)
    a.k_new = a.v_new = None
    a.tables, a.lens, a.dst = p(to["tables"]), p(to["lens"]), p(again)
    assert K.b200_paged_attn(C.byref(c.pool), C.byref(a), stream()) == 0
    torch.cuda.synchronize()
    assert status.tolist()[0] == 0 and torch.equal(again, out)
    assert set(np.flatnonzero(to["refs"].cpu().numpy())) == set(range(int((refs > 0).sum())))
