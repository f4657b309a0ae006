"""Beam search on a paged key/value cache: cases, plain forms and calls of its operators.

Five operators of the decoder side, called one after the other in every step of a beam search:

  select   the next beams over (beam, vocabulary): log-softmax, suppressed tokens, finished beams, ties to the lowest index
  reorder  per-beam state (dense caches, token histories) follows its parent beam, in place
  update   page tables of a paged cache: fork, truncate, free and grow rows; a shared page about to be written is copied
  compact  live pages move to the lowest page numbers, tables follow
  attn     a chunk of new tokens (one token included) is stored into the pages and attends over them

`run` computes them in plain torch (own = False) or through the C ABI of include/b200_whisper.h (own = True).
"""
import ctypes
import importlib.util
import math
import os
import random
import sys

import numpy as np
import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---- cases ---------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one clip decoded with 5 beams over the large vocabulary: what a single user waits for at every token
        dict(name="select 1x5 beams", op="select", n_seq=1, n_beam=5, n_vocab=51866, type="f32", banned=True, done=False),
        # 64 clips decoded together, some beams already finished, suppressed tokens as a mask
        dict(name="select 64x5 beams", op="select", n_seq=64, n_beam=5, n_vocab=51866, type="f32", banned=True, done=True),
        # dense self-attention caches of the base configuration follow their beams after 100 tokens
        dict(name="reorder base 5 beams", op="reorder", n_seq=1, n_beam=5, n_layer=6, n_ctx=448, n_past=100, dim=512),
        # the same at the large configuration: 8 clips, nearly full text context
        dict(name="reorder large 8x5 beams", op="reorder", n_seq=8, n_beam=5, n_layer=32, n_ctx=448, n_past=440, dim=1280),
        # one clip, 5 beams, large configuration: fork + one token of room + copies of the pages about to be written
        dict(name="update 1x5 beams", op="update", n_seq=1, n_beam=5, ctx=230, page=16, n_layer=32, n_kv=20, d=64, type="f16"),
        # 64 sequences of up to 4096 tokens, 5 beams each: the tables and reference counts are the work
        dict(name="update 64x5 beams long", op="update", n_seq=64, n_beam=5, ctx=4096, page=16, n_layer=1, n_kv=4, d=128, type="bf16"),
        # a small pool after a few frees
        dict(name="compact small", op="compact", n_seq=4, n_beam=1, ctx=200, page=16, n_layer=6, n_kv=8, d=64, type="f16"),
        # a large pool, half of it live and scattered
        dict(name="compact large", op="compact", n_seq=96, n_beam=1, ctx=4000, page=16, n_layer=1, n_kv=8, d=128, type="bf16"),
        # one token for each of 5 beams at the end of the text context, activations in f32 as the decoder graph has them
        dict(name="attn 5 beams 1 token f32", op="attn", n_seq=5, max_new=1, past=430, n_kv=20, group=1, d=64, type="f16", qtype="f32", page=16, ragged=False),
        # a serving batch: one token each for 64 sequences of very different lengths, grouped heads
        dict(name="attn batch 64 1 token", op="attn", n_seq=64, max_new=1, past=8191, n_kv=8, group=4, d=128, type="bf16", qtype="bf16", page=16, ragged=True),
        # prompts of 32 clips (previous text as context), every one of another length
        dict(name="attn prompts 32 ragged", op="attn", n_seq=32, max_new=224, past=0, n_kv=20, group=1, d=64, type="f16", qtype="f16", page=16, ragged=True),
        # chunked prefill deep in a long context
        dict(name="attn chunk 2048 long", op="attn", n_seq=2, max_new=2048, past=14300, n_kv=8, group=4, d=128, type="bf16", qtype="bf16", page=64, ragged=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["select", "select", "reorder", "update", "compact", "attn", "attn", "attn", "attn"])
    if op == "select":
        c = dict(op=op, n_seq=_log_int(rng, 1, 64), n_beam=rng.randint(1, 16), n_vocab=_log_int(rng, 300, 131072),
                 type=rng.choice(["f32", "f32", "f16", "bf16"]), banned=rng.random() < 0.6, done=rng.random() < 0.5)
        while c["n_seq"] * c["n_beam"] * c["n_vocab"] > 20_000_000:
            c["n_seq"] = max(1, c["n_seq"] // 2)
        return c
    if op == "reorder":
        ctx = _log_int(rng, 16, 448)
        return dict(op=op, n_seq=_log_int(rng, 1, 5), n_beam=rng.randint(2, 8), n_layer=rng.randint(1, 32), n_ctx=ctx, n_past=rng.randint(1, ctx),
                    dim=8 * rng.randint(8, 160))
    if op in ("update", "compact"):
        c = dict(op=op, n_seq=_log_int(rng, 1, 64), n_beam=rng.randint(1, 8) if op == "update" else 1, ctx=_log_int(rng, 5, 4096),
                 page=rng.choice([8, 16, 24, 32, 64]), n_layer=rng.randint(1, 8), n_kv=rng.choice([1, 2, 4, 8]), d=rng.choice([64, 128]), type=rng.choice(["f16", "bf16"]))
        while _pool_bytes(c) > 1_000_000_000:
            c["n_layer"], c["n_seq"] = (1, c["n_seq"]) if c["n_layer"] > 1 else (1, max(1, c["n_seq"] // 2))
        return c
    qtype = rng.choice(["f32", "same", "same", "same"])
    t = rng.choice(["f16", "bf16"])
    c = dict(op=op, n_seq=_log_int(rng, 1, 64), max_new=1 if rng.random() < 0.4 else _log_int(rng, 1, 2048), past=rng.choice([0, _log_int(rng, 1, 14000)]),
             n_kv=rng.choice([1, 2, 4, 8, 12, 20]), group=rng.choice([1, 1, 2, 3, 4, 5, 8]), d=rng.choice([64, 128]), type=t,
             qtype=t if qtype == "same" else qtype, page=rng.choice([5, 8, 16, 16, 32, 64, 100, 128]), ragged=rng.random() < 0.6)

    def too_much(c):
        n, heads = c["past"] + c["max_new"], c["n_kv"] * c["group"]
        flops = 4.0 * c["n_seq"] * c["max_new"] * n * heads * c["d"]
        return (flops > (2e10 if c["qtype"] == "f32" else 6e11) or 4.0 * c["n_seq"] * n * c["n_kv"] * c["d"] > 1e9
                or 4.0 * c["n_seq"] * c["max_new"] * heads * n > 6e9)

    while too_much(c):
        k = rng.choice(["n_seq", "max_new", "past"])
        c[k] = max(0 if k == "past" else 1, c[k] // 2)
    return c


def _attn_rows(c):
    """(n_new, length with the new tokens) of every sequence: fixed by the sizes, so that work() can count them."""
    r = random.Random(c["n_seq"] * 7919 + c["max_new"] * 31 + c["past"])
    rows = []
    for i in range(c["n_seq"]):
        new, past = c["max_new"], c["past"]
        if c["ragged"] and i:                      # sequence 0 has the full lengths
            new, past = r.randint(1, new), r.randint(0, past)
            if i == 1 and c["n_seq"] >= 4:
                new, past = 0, 0                   # a slot without a sequence
        rows.append((new, past + new))
    return rows


def _page_plan(c):
    """Rows of a paged cache before the call: per sequence its length, the beams' common prompt, what is kept and how many tokens come."""
    r = random.Random(c["n_seq"] * 104729 + c["n_beam"] * 1299709 + c["ctx"])
    plan = []
    for s in range(c["n_seq"]):
        length = c["ctx"] if s == 0 else r.randint(max(1, c["ctx"] // 2), c["ctx"])
        prompt = r.randint(0, length * 4 // 5) if c["n_beam"] > 1 else 0
        keep, new = length, 1
        if s and r.random() < 0.1:
            keep, new = 0, 0                       # finished: its pages are given back
        elif s and r.random() < 0.2:
            keep, new = r.randint(0, length), r.randint(0, 2 * c["page"])   # rejected tokens, then several new ones
        parents = [r.randrange(c["n_beam"]) for _ in range(c["n_beam"])]
        plan.append((length, prompt // c["page"], keep, new, parents))
    return plan


def _pages(c):
    per = [(-(-length // c["page"]), shared) for length, shared, _, _, _ in _page_plan(c)]
    used = sum(min(n, s) + c["n_beam"] * (n - min(n, s)) for n, s in per)
    rows = c["n_seq"] * c["n_beam"]
    if c["op"] == "compact":
        return used, 2 * used + 3
    return used, used + sum(max(0, -(-(k + n) // c["page"]) - k // c["page"]) * c["n_beam"] for _, _, k, n, _ in _page_plan(c)) + rows + 5


def _table_width(c):
    return -(-(c["ctx"] + 2 * c["page"] + 1) // c["page"])


def _page_bytes(c):
    return 2 * c["n_layer"] * c["page"] * c["n_kv"] * c["d"] * 2


def _pool_bytes(c):
    return _pages(c)[1] * _page_bytes(c)


# ---- inputs --------------------------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _inputs(case, seed):
    c = dict(case)
    s = {"select": _prepare_select, "reorder": _prepare_reorder, "update": _prepare_pages, "compact": _prepare_pages, "attn": _prepare_attn}[c["op"]](c, seed)
    return dict(s, case=c)


def prepare(case, seed):
    s = _inputs(case, seed)
    return dict(s, handle=_handle(s)) if own else s


def _prepare_select(c, seed):
    g, rows = _gen(seed), c["n_seq"] * c["n_beam"]
    logits = (torch.randn(rows, c["n_vocab"], generator=g, device="cuda") * 3).to(DT[c["type"]])
    score = -torch.rand(rows, generator=g, device="cuda") * 3 - 10
    done = (torch.rand(rows, generator=g, device="cuda") < 0.15).to(torch.uint8) if c["done"] else None
    words = -(-c["n_vocab"] // 32)
    banned = None
    if c["banned"]:     # about one token in eight is suppressed
        bits = [torch.randint(-2**31, 2**31 - 1, (words,), generator=g, device="cuda", dtype=torch.int32) for _ in range(3)]
        banned = bits[0] & bits[1] & bits[2]
    return dict(logits=logits, score=score, done=done, banned=banned, eos=c["n_vocab"] - 7)


def _prepare_reorder(c, seed):
    g, rows = _gen(seed), c["n_seq"] * c["n_beam"]
    k, v = (torch.randn(c["n_layer"], rows, c["n_ctx"], c["dim"], generator=g, device="cuda", dtype=torch.float16) for _ in range(2))
    hist = torch.randint(0, 51866, (rows, c["n_ctx"]), generator=g, device="cuda", dtype=torch.int32)
    parent = torch.randint(0, c["n_beam"], (rows,), generator=g, device="cuda", dtype=torch.int32)
    return dict(k=k, v=v, hist=hist, parent=parent)


def _prepare_pages(c, seed):
    g, r = _gen(seed), np.random.default_rng(seed)
    plan, (used, n_pages), width, nb = _page_plan(c), _pages(c), _table_width(c), c["n_beam"]
    rows = c["n_seq"] * nb
    ids = r.permutation(n_pages)[:used].astype(np.int32)
    tables, lens, parent, keep, new = np.full((rows, width), -1, np.int32), *(np.zeros(rows, np.int32) for _ in range(4))
    at = 0
    for s, (length, shared, k, n, parents) in enumerate(plan):
        total = -(-length // c["page"])
        shared = min(shared, total)
        mine = slice(s * nb, (s + 1) * nb)
        tables[mine, :shared] = ids[at:at + shared]
        at += shared
        own_pages = nb * (total - shared)
        tables[mine, shared:total] = ids[at:at + own_pages].reshape(nb, total - shared)
        at += own_pages
        lens[mine], keep[mine], new[mine] = length, k, n
        parent[mine] = [s * nb + p for p in parents]
    refs = np.bincount(tables[tables >= 0], minlength=n_pages).astype(np.int32)
    pool = torch.randn(2, c["n_layer"], n_pages, c["page"], c["n_kv"], c["d"], generator=g, device="cuda", dtype=DT[c["type"]])
    dev = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    s = dict(pool=pool, tables=dev(tables), lens=dev(lens), refs=dev(refs), parent=dev(parent), keep=dev(keep), new=dev(new))
    s["to"] = dict(tables=torch.empty_like(s["tables"]), lens=torch.empty_like(s["lens"]), refs=torch.empty_like(s["refs"]))
    s["status"] = torch.zeros(2, dtype=torch.int32, device="cuda")
    if c["op"] == "compact":
        s["remap"] = torch.empty(n_pages, dtype=torch.int32, device="cuda")
    return s


def _prepare_attn(c, seed):
    g, r = _gen(seed), np.random.default_rng(seed)
    rows, ps = _attn_rows(c), c["page"]
    need = [-(-n // ps) for _, n in rows]
    width, n_pages = max(need) + 1, sum(need) + 3
    ids = r.permutation(n_pages).astype(np.int32)
    tables, at = np.full((len(rows), width), -1, np.int32), 0
    for i, n in enumerate(need):
        tables[i, :n] = ids[at:at + n]
        at += n
    start = np.concatenate([[0], np.cumsum([n for n, _ in rows])]).astype(np.int32)
    n_tok, heads, d, qt = int(start[-1]), c["n_kv"] * c["group"], c["d"], DT[c["qtype"]]
    pool = torch.randn(2, n_pages, ps, c["n_kv"], d, generator=g, device="cuda", dtype=DT[c["type"]])
    q = torch.randn(n_tok, heads, d, generator=g, device="cuda", dtype=qt)
    k_new, v_new = (torch.randn(n_tok, c["n_kv"], d, generator=g, device="cuda", dtype=qt) for _ in range(2))
    dev = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    return dict(pool=pool, q=q, k_new=k_new, v_new=v_new, tables=dev(tables), lens=dev(np.array([n for _, n in rows], np.int32)), q_start=dev(start),
                max_len=max(n for _, n in rows), scale=1.0 / math.sqrt(d), out=torch.empty_like(q))


# ---- the framework's calls -----------------------------------------------------------------------------------------

def _package():
    if "whisper_cpp_b200" not in sys.modules:
        at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "whisper.cpp_b200")
        spec = importlib.util.spec_from_file_location("whisper_cpp_b200", os.path.join(at, "__init__.py"), submodule_search_locations=[at])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["whisper_cpp_b200"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["whisper_cpp_b200"]


def _p(t):
    return None if t is None else t.data_ptr()


def _handle(s):
    """The argument blocks, workspaces and output buffers that a decoding program sets up once and uses at every step."""
    P, c, op = _package(), s["case"], s["case"]["op"]
    lib, types = P.kernels_lib(), {"f32": 0, "f16": 1, "bf16": 30}
    h = {"lib": lib, "device": torch.cuda.current_device()}
    space = lambda n: torch.empty(max(int(n), 16), dtype=torch.uint8, device="cuda")  # noqa: E731
    if op == "select":
        rows = c["n_seq"] * c["n_beam"]
        h["out"] = dict(score=torch.empty(rows, device="cuda"), token=torch.empty(rows, dtype=torch.int32, device="cuda"),
                        parent=torch.empty(rows, dtype=torch.int32, device="cuda"), done=torch.empty(rows, dtype=torch.uint8, device="cuda"))
        h["ws"] = space(lib.b200_beam_select_workspace(c["n_seq"], c["n_beam"], c["n_vocab"]))
        o = h["out"]
        h["args"] = P.BeamSelectArgs(logits=_p(s["logits"]), type=types[c["type"]], nb_row=c["n_vocab"] * SIZE[c["type"]], n_vocab=c["n_vocab"], n_seq=c["n_seq"],
                                     n_beam=c["n_beam"], score=_p(s["score"]), done=_p(s["done"]), eos=s["eos"], banned=_p(s["banned"]), banned_stride=0,
                                     score_out=_p(o["score"]), token_out=_p(o["token"]), parent_out=_p(o["parent"]), done_out=_p(o["done"]),
                                     workspace=_p(h["ws"]), workspace_bytes=h["ws"].numel())
    elif op == "reorder":
        row = c["n_ctx"] * c["dim"] * 2
        rows = c["n_seq"] * c["n_beam"]
        h["args"] = (P.BeamBlock * 3)(*[P.BeamBlock(base=_p(s[n]), n_outer=c["n_layer"], nb_outer=rows * row, nb_row=row, row_bytes=c["n_past"] * c["dim"] * 2) for n in "kv"],
                                      P.BeamBlock(base=_p(s["hist"]), n_outer=1, nb_outer=0, nb_row=c["n_ctx"] * 4, row_bytes=c["n_past"] * 4))
        h["parent"] = _p(s["parent"])
    elif op in ("update", "compact"):
        n_pages, tok = s["pool"].shape[2], c["n_kv"] * c["d"] * 2
        page = c["page"] * tok
        h["pool"] = P.PagePool(k=_p(s["pool"][0]), v=_p(s["pool"][1]), type=types[c["type"]], n_layer=c["n_layer"], n_pages=n_pages, page_size=c["page"], n_head_kv=c["n_kv"],
                               head_dim=c["d"], nb_layer=n_pages * page, nb_page=page, nb_tok=tok, nb_head=c["d"] * 2)
        one = lambda t: P.PageState(tables=_p(t["tables"]), lens=_p(t["lens"]), refs=_p(t["refs"]), n_rows=s["tables"].shape[0], table_stride=s["tables"].shape[1])  # noqa: E731
        h["from"], h["to"] = one(s), one(s["to"])
        h["ws"] = space(lib.b200_pages_workspace(s["tables"].shape[0], n_pages))
    else:
        tok, new_tok = c["n_kv"] * c["d"] * 2, c["n_kv"] * c["d"] * SIZE[c["qtype"]]
        page, q_head = c["page"] * tok, c["d"] * SIZE[c["qtype"]]
        heads = c["n_kv"] * c["group"]
        h["pool"] = P.PagePool(k=_p(s["pool"][0]), v=_p(s["pool"][1]), type=types[c["type"]], n_layer=1, n_pages=s["pool"].shape[1], page_size=c["page"], n_head_kv=c["n_kv"],
                               head_dim=c["d"], nb_layer=0, nb_page=page, nb_tok=tok, nb_head=c["d"] * 2)
        a = h["args"] = P.PagedAttnArgs(q=_p(s["q"]), q_type=types[c["qtype"]], nb_q_tok=heads * q_head, nb_q_head=q_head, dst=_p(s["out"]), nb_dst_tok=heads * q_head,
                                        nb_dst_head=q_head, k_new=_p(s["k_new"]), v_new=_p(s["v_new"]), nb_new_tok=new_tok, nb_new_head=q_head, layer=0,
                                        tables=_p(s["tables"]), table_stride=s["tables"].shape[1], lens=_p(s["lens"]), q_start=_p(s["q_start"]), n_tok=s["q"].shape[0],
                                        n_seq=c["n_seq"], n_head=heads, max_new=c["max_new"], max_len=s["max_len"], causal=1, scale=s["scale"])
        h["ws"] = space(lib.b200_paged_attn_workspace(ctypes.byref(h["pool"]), ctypes.byref(a)))
        a.workspace, a.workspace_bytes = _p(h["ws"]), h["ws"].numel()
    return h


def _checked(rc):
    if rc != 0:
        raise RuntimeError("the call returned %d" % rc)


def _run_own(s):
    h, c = s["handle"], s["case"]
    op, lib, ref, stream = c["op"], h["lib"], ctypes.byref, torch._C._cuda_getCurrentRawStream(h["device"])      # as torch.cuda.current_stream().cuda_stream, 3 us less
    if op == "select":
        _checked(lib.b200_beam_select(ref(h["args"]), stream))
        return h["out"]
    if op == "reorder":
        _checked(lib.b200_beam_reorder(h["args"], 3, h["parent"], c["n_seq"], c["n_beam"], stream))
        return dict(k=s["k"], v=s["v"], hist=s["hist"])
    if op == "update":
        _checked(lib.b200_pages_update(ref(h["pool"]), ref(h["from"]), ref(h["to"]), _p(s["parent"]), _p(s["keep"]), _p(s["new"]), _p(s["status"]), _p(h["ws"]),
                                       h["ws"].numel(), stream))
        return dict(s["to"], pool=s["pool"], status=s["status"])
    if op == "compact":
        _checked(lib.b200_pages_compact(ref(h["pool"]), ref(h["from"]), ref(h["to"]), _p(s["remap"]), _p(s["status"]), _p(h["ws"]), h["ws"].numel(), stream))
        return dict(s["to"], pool=s["pool"], remap=s["remap"], status=s["status"])
    _checked(lib.b200_paged_attn(ref(h["pool"]), ref(h["args"]), stream))
    return dict(out=s["out"], pool=s["pool"])


# ---- plain forms ---------------------------------------------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    return {"select": _select, "reorder": _reorder, "update": _update, "compact": _compact, "attn": _attn}[state["case"]["op"]](state)


def _select(s):
    """score[b] + x - max - log(sum(exp(x - max))) over the allowed tokens; in 64 bits, because neighbouring candidates decide which beams live."""
    c = s["case"]
    n, b, v = c["n_seq"], c["n_beam"], c["n_vocab"]
    x = s["logits"].double()
    if s["banned"] is not None:
        at = torch.arange(v, device="cuda")
        x = x.masked_fill(((s["banned"][at // 32] >> (at % 32)) & 1).bool(), -math.inf)
    x = x - x.amax(-1, keepdim=True)
    x = x - x.exp().sum(-1, keepdim=True).log()
    cand = (x + s["score"].double()[:, None])
    if s["done"] is not None:
        only = torch.full_like(cand, -math.inf)
        only[:, s["eos"]] = s["score"].double()
        cand = torch.where(s["done"].bool()[:, None], only, cand)
    best, at = cand.view(n, b * v).sort(dim=-1, descending=True, stable=True)
    best, at = best[:, :b], at[:, :b]
    parent, token = at // v, at % v
    done = token == s["eos"]
    if s["done"] is not None:
        done = done | s["done"].view(n, b).bool().gather(1, parent)
    return dict(score=best.float().reshape(-1), token=token.int().reshape(-1), parent=parent.int().reshape(-1), done=done.to(torch.uint8).reshape(-1))


def _reorder(s):
    c = s["case"]
    rows = torch.arange(c["n_seq"] * c["n_beam"], device="cuda")
    src = rows // c["n_beam"] * c["n_beam"] + s["parent"]
    for t in (s["k"], s["v"]):
        t[:, :, :c["n_past"]] = t[:, src, :c["n_past"]]
    s["hist"][:, :c["n_past"]] = s["hist"][src, :c["n_past"]]
    return dict(k=s["k"], v=s["v"], hist=s["hist"])


def _count(ids, mask, n):
    """How often every page number occurs among `ids` where `mask` holds."""
    return torch.zeros(n + 1, dtype=torch.int32, device="cuda").index_add_(0, torch.where(mask, ids, n).reshape(-1).long(), torch.ones_like(ids).reshape(-1))[:n]


def _update(s):
    """Row i becomes the first keep[i] tokens of row parent[i] with room for new[i] more. A page that would be written and has other
    holders is copied; among several writers the first keeps the page unless somebody only reads it. Pages come lowest number first."""
    c, ps = s["case"], s["case"]["page"]
    tables, lens, refs, keep, new = s["tables"], s["lens"].long(), s["refs"], s["keep"].long(), s["new"].long()
    n_rows, width = tables.shape
    n_pages, col = refs.shape[0], torch.arange(width, device="cuda")
    src = tables[s["parent"].long()]
    kept, total = -(-keep // ps), -(-(keep + new) // ps)
    shared = col < kept[:, None]
    held = refs - _count(tables, col < (-(-lens // ps))[:, None], n_pages) + _count(src, shared, n_pages)
    writes = (keep % ps != 0) & (new > 0)
    page = torch.where(writes, src.gather(1, (keep // ps).clamp(max=width - 1)[:, None])[:, 0].long(), 0)
    same = (page[:, None] == page[None, :]) & writes[:, None] & writes[None, :]
    earlier = (same & (torch.arange(n_rows, device="cuda")[None, :] < torch.arange(n_rows, device="cuda")[:, None])).any(1)
    readers = held[page] - same.sum(1)
    copy = writes & (earlier | (readers > 0))
    first = kept - copy.long()                     # first column with a new page
    wanted = total - first
    offset = wanted.cumsum(0) - wanted
    free = (refs != 0).to(torch.uint8).sort(dim=0, stable=True).indices
    fresh = (col >= first[:, None]) & (col < total[:, None])
    number = free[(offset[:, None] + col - first[:, None]).clamp(0, n_pages - 1)].int()
    out = torch.where(fresh, number, torch.where(shared, src, -1))
    held = held - _count(page.int(), copy, n_pages) + _count(number, fresh, n_pages)
    missing = (wanted.sum() - (refs == 0).sum()).clamp(min=0)
    who = copy.nonzero()[:, 0]
    into = out.gather(1, (keep // ps).clamp(max=width - 1)[:, None])[who, 0].long()
    pool = s["pool"]
    inside = torch.arange(ps, device="cuda") < (keep % ps)[who, None]
    pool[:, :, into] = torch.where(inside[:, :, None, None], pool[:, :, page[who]], pool[:, :, into])
    s["to"]["tables"].copy_(out)
    s["to"]["lens"].copy_(keep + new)
    s["to"]["refs"].copy_(held)
    s["status"].copy_(torch.stack([missing, copy.sum()]))
    return dict(s["to"], pool=pool, status=s["status"])


def _compact(s):
    """With L live pages, the i-th live page numbered L or more moves to the i-th free page below L; tables and counts follow."""
    tables, refs, pool = s["tables"], s["refs"], s["pool"]
    n_pages, live = refs.shape[0], refs > 0
    page = torch.arange(n_pages, device="cuda")
    count = live.sum()
    away, hole = live & (page >= count), ~live & (page < count)
    src, dst = away.nonzero()[:, 0], hole.nonzero()[:, 0]
    remap = torch.where(live, page, -1)
    remap[src] = dst
    pool[:, :, dst] = pool[:, :, src]
    s["remap"].copy_(remap)
    in_use = torch.arange(tables.shape[1], device="cuda") < (-(-s["lens"].long() // s["case"]["page"]))[:, None]
    s["to"]["tables"].copy_(torch.where(in_use, remap[tables.clamp(min=0).long()], -1))
    s["to"]["lens"].copy_(s["lens"])
    held = torch.where(live, refs, 0)
    held[dst] = refs[src]
    held[src] = 0
    s["to"]["refs"].copy_(held)
    s["status"].copy_(torch.stack([torch.zeros_like(count), away.sum()]))
    return dict(s["to"], pool=pool, remap=s["remap"], status=s["status"])


def _attn(s):
    """Token t of a sequence with n_new new tokens stands at p = len - n_new + t; it is stored there and attends to positions 0 .. p."""
    c, ps, pool, lens, start = s["case"], s["case"]["page"], s["pool"], s["lens"].long(), s["q_start"].long()
    n_seq, n_kv, g, d = c["n_seq"], c["n_kv"], c["group"], c["d"]
    n_tok = s["q"].shape[0]
    tok = torch.arange(n_tok, device="cuda")
    seq = torch.searchsorted(start[1:], tok, right=True)
    t = tok - start[seq]
    pos = lens[seq] - (start[1:] - start[:-1])[seq] + t
    page = s["tables"][seq, pos // ps].long()
    pool[0][page, pos % ps] = s["k_new"].to(pool.dtype)
    pool[1][page, pos % ps] = s["v_new"].to(pool.dtype)
    n = s["max_len"]
    pages = s["tables"][:, : -(-n // ps)].long().clamp(min=0)
    k, v = (p[pages].reshape(n_seq, -1, n_kv, d)[:, :n].permute(0, 2, 1, 3).float() for p in pool)
    m = max(c["max_new"], 1)
    q = torch.zeros(n_seq, m, n_kv, g, d, device="cuda")
    q[seq, t] = s["q"].float().view(n_tok, n_kv, g, d)
    q = q.permute(0, 2, 1, 3, 4).reshape(n_seq, n_kv, m * g, d)
    w = torch.matmul(q, k.transpose(-1, -2)).mul_(s["scale"]).view(n_seq, n_kv, m, g, n)
    last = torch.full((n_seq, m), -1, device="cuda", dtype=torch.long)
    last[seq, t] = pos
    out_of_reach = torch.arange(n, device="cuda") > last[:, :, None]
    w.masked_fill_(out_of_reach[:, None, :, None, :], -math.inf)
    top = w.amax(-1, keepdim=True)
    w.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = w.sum(-1, keepdim=True)
    out = torch.matmul(w.view(n_seq, n_kv, m * g, n), v).view(n_seq, n_kv, m, g, d) / total.clamp(min=1e-30)
    s["out"].copy_(out.permute(0, 2, 1, 3, 4)[seq, t].reshape(n_tok, n_kv * g, d))
    return dict(out=s["out"], pool=pool)


# ---- 64 bits -------------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = _inputs(case, seed)
    return {"select": _exact_select, "reorder": _exact_reorder, "update": _exact_update, "compact": _exact_compact, "attn": _exact_attn}[case["op"]](s)


def _exact_select(s):
    c = s["case"]
    v, b = c["n_vocab"], c["n_beam"]
    words = None if s["banned"] is None else s["banned"].cpu().numpy().view(np.uint32)
    ok = np.ones(v, bool) if words is None else np.unpackbits(words.view(np.uint8), bitorder="little")[:v] == 0
    score, done = s["score"].double().cpu().numpy(), None if s["done"] is None else s["done"].cpu().numpy()
    res = []
    for q in range(c["n_seq"]):
        cand = []
        for j in range(b):
            row = q * b + j
            if done is not None and done[row]:
                cand.append((-score[row], j, s["eos"], 1))
                continue
            x = s["logits"][row].double().cpu().numpy()
            x[~ok] = -np.inf
            lp = x - x.max() - np.log(np.exp(x - x.max()).sum()) + score[row]
            few = np.lexsort((np.arange(v), -lp))[:b]
            cand += [(-lp[i], j, int(i), int(i == s["eos"])) for i in few]
        res += sorted(cand)[:b]
    col = lambda k, t: torch.tensor([r[k] for r in res], dtype=t)  # noqa: E731
    return dict(score=-col(0, torch.float64), token=col(2, torch.int32), parent=col(1, torch.int32), done=col(3, torch.uint8))


def _exact_reorder(s):
    c, parent = s["case"], s["parent"].tolist()
    out = {n: s[n].clone() for n in ("k", "v", "hist")}
    for row, p in enumerate(parent):
        src = row // c["n_beam"] * c["n_beam"] + p
        for n in "kv":
            out[n][:, row, :c["n_past"]] = s[n][:, src, :c["n_past"]]
        out["hist"][row, :c["n_past"]] = s["hist"][src, :c["n_past"]]
    return out


def _exact_update(s):
    c, ps = s["case"], s["case"]["page"]
    old, lens, refs = s["tables"].cpu().numpy(), s["lens"].tolist(), s["refs"].tolist()
    parent, keep, new = s["parent"].tolist(), s["keep"].tolist(), s["new"].tolist()
    free = [p for p, r in enumerate(refs) if r == 0]
    pool, tables = s["pool"].clone(), [[] for _ in parent]
    for row, n in enumerate(lens):
        for p in old[row, : -(-n // ps)]:
            refs[p] -= 1
    writers, readers = {}, {p: r for p, r in enumerate(refs) if r > 0}
    for i, p in enumerate(parent):
        tables[i] = old[p, : -(-keep[i] // ps)].tolist()
        mine = tables[i][-1] if keep[i] % ps and new[i] else None
        for x in tables[i]:
            if x == mine:
                writers.setdefault(x, []).append(i)
            else:
                readers[x] = readers.get(x, 0) + 1
    copies = 0
    for i in range(len(parent)):
        if keep[i] % ps and new[i]:
            x = tables[i][-1]
            if x in readers or writers[x][0] != i:
                y = free.pop(0)
                pool[:, :, y, : keep[i] % ps] = s["pool"][:, :, x, : keep[i] % ps]
                tables[i][-1] = y
                copies += 1
        while len(tables[i]) * ps < keep[i] + new[i]:
            tables[i].append(free.pop(0))
    held = list(refs)
    for t in tables:
        for x in t:
            held[x] += 1
    width = old.shape[1]
    i32 = lambda a: torch.tensor(a, dtype=torch.int32)  # noqa: E731
    return dict(tables=i32([t + [-1] * (width - len(t)) for t in tables]), lens=i32([a + b for a, b in zip(keep, new)]), refs=i32(held), pool=pool, status=i32([0, copies]))


def _exact_compact(s):
    refs, lens, ps = s["refs"].tolist(), s["lens"].tolist(), s["case"]["page"]
    live = [p for p, r in enumerate(refs) if r > 0]
    holes, where, moves = iter([p for p in range(len(live)) if refs[p] == 0]), {}, []
    for p in live:
        where[p] = p if p < len(live) else next(holes)
        if where[p] != p:
            moves.append((p, where[p]))
    pool = s["pool"].clone()
    if moves:
        a, b = (torch.tensor(x, device="cuda") for x in zip(*moves))
        pool[:, :, b] = s["pool"][:, :, a]
    old = s["tables"].cpu().numpy()
    width = old.shape[1]
    tables = [[where[int(x)] for x in old[i, : -(-n // ps)]] for i, n in enumerate(lens)]
    held = [0] * len(refs)
    for p in live:
        held[where[p]] = refs[p]
    i32 = lambda a: torch.tensor(a, dtype=torch.int32)  # noqa: E731
    return dict(tables=i32([t + [-1] * (width - len(t)) for t in tables]), lens=i32(lens), refs=i32(held), pool=pool,
                remap=i32([where.get(p, -1) for p in range(len(refs))]), status=i32([0, len(moves)]))


def _exact_attn(s):
    c, ps, g = s["case"], s["case"]["page"], s["case"]["group"]
    pool, out, at = s["pool"].clone(), torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    for i, (n_new, n) in enumerate(_attn_rows(c)):
        if n_new == 0:
            continue
        pages, mine = s["tables"][i].long(), slice(at, at + n_new)
        at += n_new
        where = torch.arange(n - n_new, n, device="cuda")
        pool[0, pages[where // ps], where % ps] = s["k_new"][mine].to(pool.dtype)
        pool[1, pages[where // ps], where % ps] = s["v_new"][mine].to(pool.dtype)
        everyone = torch.arange(n, device="cuda")
        for h in range(c["n_kv"]):
            k, v = (p[pages[everyone // ps], everyone % ps, h].double() for p in pool)
            for j in range(h * g, (h + 1) * g):
                w = s["q"][mine, j].double() @ k.T * s["scale"]
                w = torch.softmax(torch.where(everyone[None, :] <= where[:, None], w, -math.inf), -1)
                out[mine, j] = w @ v
    return dict(out=out, pool=pool)


# ---- work ----------------------------------------------------------------------------------------------------------

def work(case):
    c, op = case, case["op"]
    if op == "select":
        rows, size = c["n_seq"] * c["n_beam"], SIZE[c["type"]]
        live = 0.85 if c["done"] else 1.0
        return {"bytes": rows * live * c["n_vocab"] * size + rows * 20 + (c["n_vocab"] / 8 if c["banned"] else 0), "flops": rows * live * c["n_vocab"] * 4}
    if op == "reorder":
        # a row that follows itself moves nothing; of the others each distinct parent is read once and each follower written
        rows, b = c["n_seq"] * c["n_beam"], c["n_beam"]
        written = 1 - 1 / b
        read = 1 - (1 - 1 / b) ** (b - 1)
        return {"bytes": rows * (written + read) * c["n_past"] * (2 * c["n_layer"] * c["dim"] * 2 + 4), "flops": 0}
    if op in ("update", "compact"):
        plan, (used, n_pages), rows = _page_plan(c), _pages(c), c["n_seq"] * c["n_beam"]
        meta = sum(c["n_beam"] * -(-p[0] // c["page"]) * 4 * 2 for p in plan) + rows * _table_width(c) * 4 + n_pages * 8 + rows * 20
        if op == "compact":
            return {"bytes": meta + n_pages * 4 + 2 * used * (1 - used / n_pages) * _page_bytes(c), "flops": 0}
        copied = 0
        for length, shared, keep, new, parents in plan:
            if keep % c["page"] and new:
                copied += (c["n_beam"] - len(set(parents))) * (keep % c["page"]) / c["page"]
        return {"bytes": meta + 2 * copied * _page_bytes(c), "flops": 0}
    heads, moved, flops = c["n_kv"] * c["group"], 0, 0
    for n_new, n in _attn_rows(c):
        moved += 2 * (n - n_new) * c["n_kv"] * c["d"] * 2 + 2 * n_new * c["n_kv"] * c["d"] * (SIZE[c["qtype"]] + 2) + 2 * n_new * heads * c["d"] * SIZE[c["qtype"]]
        flops += 4 * heads * c["d"] * (n_new * (n - n_new) + n_new * (n_new + 1) / 2)
    return {"bytes": moved, "flops": flops}
