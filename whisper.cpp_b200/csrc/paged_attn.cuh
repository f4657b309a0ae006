// What the kernels of attention over a paged cache share (k_paged_attn.cu, k_paged_attn_tc.cu).
#pragma once
#include "b200_common.cuh"
#include <cuda_bf16.h>

struct PaArgs {
    const char * q; int64_t nb_q_tok, nb_q_head;
    char * dst; int64_t nb_dst_tok, nb_dst_head;
    const char * k; const char * v; int64_t nb_page, nb_tok, nb_head;
    const int32_t * tables; int64_t table_stride; const int32_t * lens; const int32_t * q_start; const int32_t * status;
    float * lse;
    float * part;                   // partial rows: head_dim sums, maximum, sum of weights, pad (head_dim + 4 floats)
    int64_t n_tok, max_len;
    int n_pages, page_size, n_head, n_head_kv, group, max_new, causal, n_split, chunk, tile_rows, stream, n_seq, tiles, n_whole;
    float scale_log2;               // scale * log2(e): weights are powers of two
    int early;                      // the launch before this one is the store of the same call: what it waited for is there
};

// 2^x; below 2^-126 it is 0
__device__ __forceinline__ float pa_exp2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

// not 0: the state has no room for the new tokens, and the call does nothing.  Asked for once a kernel, ahead of the loads of the first sequence, and looked
// at behind them (as a part of pa_seq: 5 beams of 431 keys 9.1 -> 9.4 us, chunks of 1024 f32 queries 1548 -> 1593)
__device__ __forceinline__ int pa_failed(const PaArgs & a) { return a.status ? *a.status : 0; }

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

// How the tcgen05 form (k_paged_attn_tc.cu) deals out its items (sequence, key/value head, tile; `tiles` per head, in this order): one CTA each for
// the first n_whole, which fill the device a whole number of times, and n_split CTAs with `chunk` keys each for those that are left, so
// that the last wave is as full as the others (chunk of 2048 over 16k keys, 512 items on 148 SMs: 3.5 waves instead of 4).  Neighbouring CTAs are
// tiles of one head and read the same keys at about the same time, from L2.
struct PaItem { int seq, kvh, tile, split; int64_t slot; };         // split: -1 = whole; slot: of its part, in tiles
__device__ __forceinline__ PaItem pa_item(const PaArgs & a, unsigned cta) {
    PaItem p;
    unsigned i = cta;
    p.split = -1; p.slot = 0;
    if (cta >= (unsigned) a.n_whole) {
        const unsigned k = cta - a.n_whole;
        i = a.n_whole + k / a.n_split;
        if (a.n_split > 1) { p.split = k % a.n_split; p.slot = k; }
    }
    const unsigned head = i / a.tiles;
    p.tile = a.tiles - 1 - (i - head * a.tiles);                   // the longest tiles first
    p.seq = head / a.n_head_kv;
    p.kvh = head - p.seq * a.n_head_kv;
    return p;
}

// rows of a tile, keys of a block, CTAs on an SM
#define PA_TC_ROWS(head_dim) ((head_dim) == 64 ? 128 : 256)
#define PA_TC_KEYS(head_dim) ((head_dim) == 64 ? 64 : 128)
#define PA_TC_CTAS(head_dim) ((head_dim) == 64 ? 4 : 1)
cudaError_t pa_tc_launch(const PaArgs & a, int head_dim, int type, int64_t n_items, cudaStream_t st);
