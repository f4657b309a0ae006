// What the kernels of attention over a paged cache share (k_paged_attn.cu, k_paged_attn_tc.cu).
#pragma once
#include "b200_common.cuh"
#include <cuda_bf16.h>

struct PaArgs {
    const char * q; int64_t nb_q_tok, nb_q_head;
    char * dst; int64_t nb_dst_tok, nb_dst_head;
    const char * k; const char * v; int64_t nb_page, nb_tok, nb_head;
    const int32_t * tables; int64_t table_stride; const int32_t * lens; const int32_t * q_start;
    float * lse;
    float * part;                   // partial rows: head_dim sums, maximum, sum of weights, pad (head_dim + 4 floats)
    int64_t n_tok, max_len;
    int n_pages, page_size, n_head, n_head_kv, group, max_new, causal, tile_rows, stream, whole, n_seq;
    float scale_log2;               // scale * log2(e): weights are powers of two
};

// 2^x; below 2^-126 it is 0
__device__ __forceinline__ float pa_exp2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

// the sequence's tokens: first query token, number of queries, keys in the pages (all cut to what the host was told)
struct PaSeq { int64_t tok0; int n_new, len; };
__device__ __forceinline__ PaSeq pa_seq(const PaArgs & a, int s) {
    PaSeq r;
    const int64_t b = a.q_start[s], e = a.q_start[s + 1];
    r.tok0 = b;
    const int64_t n = (b < 0 || e > a.n_tok || e < b) ? 0 : e - b;
    r.n_new = (int) (n < a.max_new ? n : a.max_new);
    int64_t len = a.lens[s];
    len = len < 0 ? 0 : len < a.max_len ? len : a.max_len;
    const int64_t room = a.table_stride * a.page_size;
    r.len = (int) (len < room ? len : room);
    return r;
}

// keys that any row of the tile (tile_rows rows, row0 the first) sees, from the first key
__device__ __forceinline__ int pa_reach(const PaArgs & a, const PaSeq & s, int row0) {
    const int last_t = (min(row0 + a.tile_rows, s.n_new * a.group) - 1) / a.group;
    return a.causal ? min(s.len, max(s.len - s.n_new + last_t + 1, 0)) : s.len;
}

// How the work is dealt out.  Items are (sequence, key/value head, tile of tile_rows rows), numbered in that order; an item of a sequence of
// n keys is ceil(n / round) rounds of `round` keys, at least one.  Either a CTA takes one item (stream = 0), or the rounds of all items are
// one line that is cut into `stream` equal parts, one per CTA: whatever the lengths, all CTAs end together.  On the line an item begins with
// PA_START steps of nothing, the time that it takes to get its first keys (one token for 64 sequences of 1 to 8192 keys: 224 us without it,
// 183 with 2, 181 with 4 or 8).  A CTA then has up to two partial items, at the ends of its part; it leaves them in slots 0 (an item begun
// by another CTA) and 1, and k_paged_join puts them together.  That the first tiles of a chunk reach fewer keys is not on the line: sums over
// the tiles would cost every CTA more than the evenness gains.
// Tiles of one head that run side by side read the same keys at about the same time, from L2; dealt out as one line they would not (chunk of
// 2048 over 16k keys, 134 MB of K and V: 1.31 ms instead of 1.15).  So where there are more items than CTAs (whole = 1), CTA c first takes
// items c, c + stream, .. as long as every CTA gets one, and only the rest is a line.
#define PA_START 3
__device__ __forceinline__ int pa_tiles(const PaArgs & a, const PaSeq & s) { return (s.n_new * a.group + a.tile_rows - 1) / a.tile_rows; }
__device__ __forceinline__ int64_t pa_items(const PaArgs & a, const PaSeq & s) { return (int64_t) pa_tiles(a, s) * a.n_head_kv; }
__device__ __forceinline__ int pa_steps(const PaSeq & s, int round) { return max(1, (s.len + round - 1) / round) + PA_START; }      // of an item

// Sums over the sequences are a warp's: its lanes take a run of them each.
struct PaRuns { int s0, s1; int64_t before, total; };      // this lane's sequences; the sum over those before, and over all
template <typename F>
__device__ __forceinline__ PaRuns pa_runs(const PaArgs & a, F of) {
    const int lane = threadIdx.x & 31, per = (a.n_seq + 31) / 32;
    PaRuns r;
    r.s0 = min(a.n_seq, lane * per); r.s1 = min(a.n_seq, r.s0 + per);
    int64_t mine = 0;
    for (int s = r.s0; s < r.s1; ++s) mine += of(s, pa_seq(a, s));
    int64_t inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int64_t u = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += u; }
    r.before = inc - mine;
    r.total = __shfl_sync(0xffffffffu, inc, 31);
    return r;
}
// the sequence that holds place w of the sum, and how far in it w is; n_seq if none does
template <typename F>
__device__ __forceinline__ int pa_place(const PaArgs & a, const PaRuns & r, int64_t w, F of, int64_t * rest) {
    int s = r.s0;
    int64_t left = w - r.before;
    bool here = false;
    if (left >= 0) for (; s < r.s1; ++s) { const int64_t n = of(s, pa_seq(a, s)); if (left < n) { here = true; break; } left -= n; }
    const unsigned who = __ballot_sync(0xffffffffu, here);
    const int src = who ? __ffs(who) - 1 : 0;
    *rest = __shfl_sync(0xffffffffu, left, src);
    s = __shfl_sync(0xffffffffu, s, src);
    return who ? s : a.n_seq;
}

// The line: its steps, its first item (sequence, item of the sequence), whole items per CTA before it.  All lanes of a warp together.
struct PaLine { int64_t total; int seq0; int64_t item0; int64_t whole; PaRuns runs; };
__device__ __forceinline__ int64_t pa_on_line(const PaArgs & a, const PaLine & l, int round, int i, const PaSeq & s) {      // steps of a sequence
    return i < l.seq0 ? 0 : (pa_items(a, s) - (i == l.seq0 ? l.item0 : 0)) * pa_steps(s, round);
}
__device__ __forceinline__ PaLine pa_line(const PaArgs & a, int round) {
    PaLine l = {};
    if (a.whole) {
        auto items = [&](int, const PaSeq & s) { return pa_items(a, s); };
        const PaRuns r = pa_runs(a, items);
        l.whole = r.total / a.stream;
        l.seq0 = pa_place(a, r, l.whole * a.stream, items, &l.item0);
    }
    l.runs = pa_runs(a, [&](int i, const PaSeq & s) { return pa_on_line(a, l, round, i, s); });
    l.total = l.runs.total;
    return l;
}
// the item that holds place w of the line, and how far in it w is; seq = n_seq if none does
struct PaPlace { int seq, kvh, tile, at; };
__device__ __forceinline__ PaPlace pa_locate(const PaArgs & a, int round, const PaLine & l, int64_t w) {
    PaPlace p = { 0, 0, 0, 0 };
    int64_t rest;
    p.seq = pa_place(a, l.runs, w, [&](int i, const PaSeq & s) { return pa_on_line(a, l, round, i, s); }, &rest);
    if (p.seq >= a.n_seq) return p;
    const PaSeq s = pa_seq(a, p.seq);
    const int steps = pa_steps(s, round), tiles = pa_tiles(a, s);
    const int64_t item = rest / steps;
    p.at = (int) (rest - item * steps);
    const unsigned i = (unsigned) (item + (p.seq == l.seq0 ? l.item0 : 0));       // at most 64 tiles of 1024 heads
    p.kvh = (int) (i / (unsigned) tiles);
    p.tile = (int) (i - p.kvh * (unsigned) tiles);
    return p;
}

#define PA_WHOLE 8             // whole items of a CTA, at most
struct PaDealer { int seq, kvh, tile, at, n_whole; int64_t todo; };   // the next item, where on the line in it, what is left of this CTA's part
struct PaItem { int seq, kvh, tile; };
struct PaSeg { PaSeq s; int seq, kvh, tile, row0, n_rows, k0, k1; bool whole; };      // keys k0 .. k1-1 of an item; whole: all that it has
// All lanes of a warp together, the same in every warp; false: nothing to do.  items: room for PA_WHOLE items, written by every warp with the
// same values (whole items only).
__device__ __forceinline__ bool pa_deal_init(const PaArgs & a, int round, PaDealer & d, PaItem * items) {
    d.todo = 1; d.at = 0; d.n_whole = 0;
    if (!a.stream) { d.seq = blockIdx.z; d.kvh = blockIdx.y; d.tile = gridDim.x - 1 - blockIdx.x; return true; }      // the longest tiles first
    const PaLine l = pa_line(a, round);
    if (a.whole) {
        auto of = [&](int, const PaSeq & s) { return pa_items(a, s); };
        const PaRuns r = pa_runs(a, of);
        d.n_whole = (int) min(l.whole, (int64_t) PA_WHOLE);
        for (int i = 0; i < d.n_whole; ++i) {
            int64_t rest;
            const int seq = pa_place(a, r, blockIdx.x + (int64_t) i * a.stream, of, &rest);
            const unsigned tiles = max(1, pa_tiles(a, pa_seq(a, min(seq, a.n_seq - 1)))), item = (unsigned) rest;
            items[i].seq = seq; items[i].kvh = item / tiles; items[i].tile = item % tiles;
        }
    }
    const int64_t w = blockIdx.x * l.total / a.stream;
    d.todo = ((int64_t) blockIdx.x + 1) * l.total / a.stream - w;
    const PaPlace p = pa_locate(a, round, l, w);
    d.seq = p.seq; d.kvh = p.kvh; d.tile = p.tile; d.at = p.at;
    if (p.seq >= a.n_seq) d.todo = 0;
    return d.todo > 0 || d.n_whole > 0;
}
// the next piece of work of this CTA; false: no more
__device__ __forceinline__ bool pa_deal_next(const PaArgs & a, int round, PaDealer & d, PaSeg & g, const PaItem * items, int * taken) {
    if (*taken < d.n_whole) {
        const PaItem i = items[(*taken)++];
        g.s = pa_seq(a, i.seq);
        g.seq = i.seq; g.kvh = i.kvh; g.tile = i.tile; g.row0 = i.tile * a.tile_rows; g.n_rows = g.s.n_new * a.group;
        g.k0 = 0; g.k1 = pa_reach(a, g.s, g.row0); g.whole = true;
        return true;
    }
    for (;;) {
        if (d.todo == 0) return false;
        g.s = pa_seq(a, d.seq);
        g.seq = d.seq; g.kvh = d.kvh; g.tile = d.tile; g.row0 = d.tile * a.tile_rows; g.n_rows = g.s.n_new * a.group;
        if (!a.stream) {
            d.todo = 0;
            g.k0 = 0; g.k1 = g.row0 < g.n_rows ? pa_reach(a, g.s, g.row0) : 0; g.whole = true;
            return g.row0 < g.n_rows;
        }
        const int all = pa_steps(g.s, round), steps = (int) min((int64_t) (all - d.at), d.todo);
        const int first = max(0, d.at - PA_START), n = max(0, d.at + steps - PA_START) - first;
        g.k0 = first * round; g.k1 = min(pa_reach(a, g.s, g.row0), g.k0 + n * round); g.whole = n == all - PA_START;
        d.todo -= steps;
        d.at = 0;
        if (d.todo > 0 && ++d.tile * a.tile_rows >= g.n_rows) {
            d.tile = 0;
            if (++d.kvh == a.n_head_kv) {
                d.kvh = 0;
                do { if (++d.seq >= a.n_seq) { d.todo = 0; break; } } while (pa_seq(a, d.seq).n_new == 0);
            }
        }
        if (n > 0) return true;
    }
}

// the tcgen05 form (k_paged_attn_tc.cu): rows of a tile, keys of a round, CTAs on an SM
#define PA_TC_ROWS(head_dim) ((head_dim) == 64 ? 128 : 256)
#define PA_TC_KEYS(head_dim) ((head_dim) == 64 ? 64 : 128)
#define PA_TC_CTAS(head_dim) ((head_dim) == 64 ? 4 : 1)
cudaError_t pa_tc_launch(const PaArgs & a, int head_dim, int type, int n_seq, cudaStream_t st);
