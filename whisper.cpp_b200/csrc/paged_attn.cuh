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
    int n_pages, page_size, n_head, n_head_kv, group, max_new, causal, tile_rows, stream, n_seq;
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

// How the work is dealt out.  Items are (sequence, key/value head, tile of tile_rows rows), numbered in that order; an item is as many rounds
// of `round` keys as its rows reach, at least one.  Either a CTA takes one item (stream = 0), or the rounds of all items are one line that
// is cut into `stream` equal parts, one per CTA: whatever the lengths, all CTAs end together.  On the line an item begins with PA_START
// steps of nothing, the time that it takes to get its first keys (one token for 64 sequences of 1 to 8192 keys: 224 us without it, 183
// with 2, 181 with 4 or 8).  A CTA then has up to two partial items, at the ends of its part; it leaves them in slots 0 (an item begun by
// another CTA) and 1, and k_paged_join puts them together.
#define PA_START 3
struct PaLine { int64_t total, before; };                 // steps of all sequences, and of those before a given one
__device__ __forceinline__ int pa_tiles(const PaArgs & a, const PaSeq & s) { return (s.n_new * a.group + a.tile_rows - 1) / a.tile_rows; }
__device__ __forceinline__ int pa_tile_steps(const PaArgs & a, const PaSeq & s, int tile, int round) {
    return max(1, (pa_reach(a, s, tile * a.tile_rows) + round - 1) / round) + PA_START;
}
__device__ __forceinline__ int64_t pa_head_steps(const PaArgs & a, const PaSeq & s, int round) {      // of all tiles of a key/value head
    int64_t n = 0;
    const int tiles = pa_tiles(a, s);
    for (int t = 0; t < tiles; ++t) n += pa_tile_steps(a, s, t, round);
    return n;
}
// this warp's lanes go over the sequences, a run of them each
__device__ __forceinline__ PaLine pa_line(const PaArgs & a, int round, int64_t cta, int upto, int * seq_at, int64_t * rest) {
    const int lane = threadIdx.x & 31, per = (a.n_seq + 31) / 32, s0 = min(a.n_seq, lane * per), s1 = min(a.n_seq, s0 + per);
    int64_t mine = 0;
    for (int s = s0; s < s1; ++s) mine += a.n_head_kv * pa_head_steps(a, pa_seq(a, s), round);
    int64_t inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int64_t u = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += u; }
    PaLine l;
    l.total = __shfl_sync(0xffffffffu, inc, 31);
    l.before = 0;
    if (upto >= 0) {                                       // steps before sequence `upto`
        int64_t b = inc - mine;
        if (upto >= s0 && upto < s1) for (int s = s0; s < upto; ++s) b += a.n_head_kv * pa_head_steps(a, pa_seq(a, s), round);
        l.before = __shfl_sync(0xffffffffu, b, upto / per);
    }
    if (seq_at) {                                          // the sequence in which CTA `cta` begins, and how far
        const int64_t w = cta * l.total / a.stream;
        const bool here = w >= inc - mine && w < inc;
        int s = s0;
        int64_t left = w - (inc - mine);
        if (here) for (; s < s1; ++s) { const int64_t r = a.n_head_kv * pa_head_steps(a, pa_seq(a, s), round); if (left < r) break; left -= r; }
        const unsigned who = __ballot_sync(0xffffffffu, here);
        const int src = who ? __ffs(who) - 1 : 0;
        *seq_at = who ? __shfl_sync(0xffffffffu, s, src) : a.n_seq;
        *rest = __shfl_sync(0xffffffffu, left, src);
    }
    return l;
}

struct PaDealer { int seq, kvh, tile, at; int64_t todo; };            // the next item, where on the line in it, what is left of this CTA's part
struct PaSeg { PaSeq s; int seq, kvh, tile, row0, n_rows, k0, k1; bool whole; };      // keys k0 .. k1-1 of an item; whole: all that it has
// all lanes of a warp together; false: nothing to do
__device__ __forceinline__ bool pa_deal_init(const PaArgs & a, int round, PaDealer & d) {
    d.todo = 1; d.at = 0;
    if (!a.stream) { d.seq = blockIdx.z; d.kvh = blockIdx.y; d.tile = gridDim.x - 1 - blockIdx.x; return true; }      // the longest tiles first
    int64_t rest;
    const PaLine l = pa_line(a, round, blockIdx.x, -1, &d.seq, &rest);
    d.todo = ((int64_t) blockIdx.x + 1) * l.total / a.stream - (int64_t) blockIdx.x * l.total / a.stream;
    if (d.seq >= a.n_seq || d.todo == 0) return false;
    const PaSeq s = pa_seq(a, d.seq);
    const int64_t head = pa_head_steps(a, s, round);
    d.kvh = (int) (rest / head);
    rest -= d.kvh * head;
    for (d.tile = 0;; ++d.tile) { const int n = pa_tile_steps(a, s, d.tile, round); if (rest < n) break; rest -= n; }
    d.at = (int) rest;
    return true;
}
// the next piece of work of this CTA; false: no more
__device__ __forceinline__ bool pa_deal_next(const PaArgs & a, int round, PaDealer & d, PaSeg & g) {
    for (;;) {
        if (d.todo == 0) return false;
        g.s = pa_seq(a, d.seq);
        g.seq = d.seq; g.kvh = d.kvh; g.tile = d.tile; g.row0 = d.tile * a.tile_rows; g.n_rows = g.s.n_new * a.group;
        if (!a.stream) {
            d.todo = 0;
            g.k0 = 0; g.k1 = g.row0 < g.n_rows ? pa_reach(a, g.s, g.row0) : 0; g.whole = true;
            return g.row0 < g.n_rows;
        }
        const int all = pa_tile_steps(a, g.s, d.tile, round), steps = (int) min((int64_t) (all - d.at), d.todo);
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
