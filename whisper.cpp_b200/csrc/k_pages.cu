// A paged key/value cache: who holds which page (fork, truncate, free, grow, compact) and the copies that follow from it.
// Counterpart in the reference: the cells of whisper_kv_cache (whisper_kv_cache_find_slot / _seq_cp / _seq_rm,
// src/whisper.cpp:1000-1200), which are host code over one dense cache.
#include "b200_common.cuh"
#include <cooperative_groups.h>
namespace cg = cooperative_groups;

// ---- copies --------------------------------------------------------------------------------------
// CTA `me` of `ctas` takes its share of (copy, layer, K or V, tile of 16-byte vectors).  Bound by memory for long lists: the bytes are read
// once and written once.
#define PG_COPY_THREADS 256
#define PG_COPY_UNROLL  4
template <typename LIST>
__device__ __forceinline__ void pg_copy(const b200_page_pool & pool, int n, int64_t me, int64_t ctas, LIST list) {
    const unsigned vec_head = pool.head_dim / 8, vec_tok = vec_head * pool.n_head_kv, vec_page = vec_tok * pool.page_size;
    const unsigned tiles = (vec_page + PG_COPY_THREADS * PG_COPY_UNROLL - 1) / (PG_COPY_THREADS * PG_COPY_UNROLL);
    const int64_t items = (int64_t) n * pool.n_layer * 2 * tiles;
    const int64_t row = pool.head_dim * 2;
    const bool toks = (pool.n_head_kv == 1 || pool.nb_head == row) && (pool.page_size == 1 || pool.nb_tok == row * pool.n_head_kv);
    const bool heads = (pool.page_size == 1 || pool.nb_tok == row) && (pool.n_head_kv == 1 || pool.nb_head == row * pool.page_size);
    for (int64_t it = me; it < items; it += ctas) {
        int64_t r = it;
        const unsigned tile = (unsigned) (r % tiles); r /= tiles;
        const int kv = (int) (r & 1); r >>= 1;
        const int layer = (int) (r % pool.n_layer);
        int src, dst, tokens;
        list(r / pool.n_layer, src, dst, tokens);
        const unsigned used = tokens * vec_tok;
        if (src < 0 || dst < 0 || src >= pool.n_pages || dst >= pool.n_pages || tokens < 0 || tokens > pool.page_size) continue;
        char * base = (char *) (kv ? pool.v : pool.k) + layer * pool.nb_layer;
        const bool flat = toks || (heads && used == vec_page);      // what is copied is one piece of memory
        uint4 v[PG_COPY_UNROLL];
        int64_t off[PG_COPY_UNROLL];
#pragma unroll
        for (int u = 0; u < PG_COPY_UNROLL; ++u) {
            const unsigned x = (tile * PG_COPY_UNROLL + u) * PG_COPY_THREADS + threadIdx.x;
            off[u] = -1;
            if (x < used && flat) {
                off[u] = x * 16ll;
                v[u] = *(const uint4 *) (base + src * pool.nb_page + off[u]);
            } else if (x < used) {
                // token-major pages: consecutive vectors walk the heads of a token; head-major: the tokens of a head come first
                // in memory, so they are walked first
                unsigned tok, h, i;
                if (pool.nb_tok >= pool.nb_head) { tok = x / vec_tok; const unsigned y = x - tok * vec_tok; h = y / vec_head; i = y - h * vec_head; }
                else { const unsigned per = tokens * vec_head; h = x / per; const unsigned y = x - h * per; tok = y / vec_head; i = y - tok * vec_head; }
                off[u] = tok * pool.nb_tok + h * pool.nb_head + i * 16;
                v[u] = *(const uint4 *) (base + src * pool.nb_page + off[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < PG_COPY_UNROLL; ++u) if (off[u] >= 0) *(uint4 *) (base + dst * pool.nb_page + off[u]) = v[u];
    }
}

// ---- tables and reference counts -----------------------------------------------------------------
// The steps depend on one another (counts -> who must copy -> which pages are taken), so all of them run in one launch.  A state that
// fits shared memory (SMALL) is loaded once and worked on there; what bounds it is the latency of that load.  Up to PG_FUSED words of
// state, every CTA of the launch does that for itself - the result is the same everywhere, CTA 0 writes it down - and then makes its share of
// the page copies: one launch and no wait for a list.  A larger small state is the work of one CTA, and the copies are a launch of their
// own.  A state that does not fit is the work of one cluster of CTAs on global memory: the hardware barrier of a cluster between the steps costs a fraction of a
// launch.  All results are integers and independent of the order of the atomics; ranks come from prefix sums.
#define PG_THREADS 1024
#define PG_CLUSTER 16
#define PG_MAX_ROWS 8192
#define PG_MAX_PAGES (1 << 30)    // so that 3 words a copy (of at most half of them) and a thread's run of pages stay within 31 bits
#define PG_SMALL   (160 * 1024)   // bytes of shared memory that a small state may take
#define PG_FUSED   3000           // words of tables and counts up to which every CTA works them out for itself (5 beams, pages of 16, 8 layers of 20 heads; us
                                  // with and without: 1 sequence of 230 tokens 7.5, 9.1; 8 of 400 10.4, 11.4; 16 of 400 16.4, 15.7; 24 of 400 19.3, 17.5)
#define PG_HEADER  8              // workspace words before the lists: [0] copies, [2] see k_pages_compact

struct PgWork { int32_t * head; int32_t * copies; int32_t * a; int32_t * b; };    // copies: (src, dst, tokens) each

static inline int64_t pg_layout(PgWork * w, void * base, int64_t n_rows, int64_t n_pages) {
    const int64_t n = n_rows > n_pages ? n_rows : n_pages;
    int32_t * p = (int32_t *) base;
    w->head = p;            p += PG_HEADER;
    w->copies = p;          p += 3 * n;
    w->a = p;               p += n;
    w->b = p;               p += n;
    return (char *) p - (char *) base;
}

struct PgState { int32_t * tables; int32_t * lens; int32_t * refs; };

// exclusive prefix sum over the block; s_warp: 32 words
template <typename V>
__device__ __forceinline__ V pg_scan(V v, V * s_warp, V * total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    V inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const V u = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += u; }
    __syncthreads();                                   // s_warp may still be read from the scan before
    if (lane == 31) s_warp[warp] = inc;
    __syncthreads();
    // every warp adds up the warps before it
    V y = lane < (int) (blockDim.x >> 5) ? s_warp[lane] : 0;
    const V mine = y;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const V u = __shfl_up_sync(0xffffffffu, y, o); if (lane >= o) y += u; }
    *total = __shfl_sync(0xffffffffu, y, 31);
    return __shfl_sync(0xffffffffu, y - mine, warp) + inc - v;
}

__device__ __forceinline__ int pg_ceil(int n, int ps) { return n / ps + (n % ps != 0); }

struct PgShared { long long warp2[32]; int warp[32]; int n; int err; };

// barrier over all threads of the launch
template <bool SMALL> __device__ __forceinline__ void pg_sync(cg::cluster_group & cl) { if (SMALL) __syncthreads(); else cl.sync(); }
// a word that another thread of the launch has written
template <bool SMALL> __device__ __forceinline__ int pg_get(const int32_t * p) { return SMALL ? *p : __ldcg(p); }

// barrier; this CTA's contribution -> sum over the CTAs before it, and over all (reads the others' shared memory: barriers around it)
template <bool SMALL>
__device__ __forceinline__ void pg_across(cg::cluster_group & cl, PgShared & s, int * before, int * all, int * err) {
    pg_sync<SMALL>(cl);
    int b = 0, t = 0, e = 0;
    if (SMALL) { t = s.n; e = s.err; }
    else {                                              // lane r asks CTA r (at most 16 of them)
        const unsigned lane = threadIdx.x & 31, me = cl.block_rank();
        int v = 0;
        if (lane < cl.num_blocks()) { const PgShared * o = cl.map_shared_rank(&s, lane); v = o->n; e = o->err; }
        e = __any_sync(0xffffffffu, e);
        t = __reduce_add_sync(0xffffffffu, v);
        b = __reduce_add_sync(0xffffffffu, lane < me ? v : 0);
    }
    *before = b; *all = t; *err = e;
}

// Loops over the cells of all tables and over a thread's run of pages load PG_BATCH values before they use the first: what they store may alias
// what they load as far as the compiler knows, and one value at a time costs a latency each (64 x 5 rows of 259 pages: 23 us).
#define PG_BATCH 4

// words of shared memory that a small state takes: tables, counts (as they are, and worked on), two lists of pages, columns of rows, copies
#define PG_COLUMNS 7
static inline int64_t pg_small_words(int64_t n_rows, int64_t width, int64_t n_pages) { return n_rows * width + 4 * n_pages + (PG_COLUMNS + 3) * n_rows; }

template <bool SMALL>
__global__ void __launch_bounds__(PG_THREADS)
k_pages_update(PgState from, PgState to, int n_rows, int width, int n_pages, int ps,
               const int32_t * parent, const int32_t * keep, const int32_t * n_new, int32_t * status, PgWork w, const __grid_constant__ b200_page_pool pool, bool fused) {
    cg::cluster_group cl = cg::this_cluster();
    __shared__ PgShared sh;
    extern __shared__ int32_t s_dyn[];
    // per row, in every CTA: its parent; pages it had, keeps, will have; its length; tokens in its last kept page if that
    // will be written, else 0, and that page; pages wanted by the rows before it (top bit: its last kept page is copied)
    int32_t * s_par = s_dyn, * s_old = s_par + n_rows, * s_kept = s_old + n_rows, * s_tot = s_kept + n_rows, * s_len = s_tot + n_rows, * s_mod = s_len + n_rows,
            * s_off = s_mod + n_rows, * s_raw = s_off, * s_page = s_old;     // the length as it was is needed only before the offsets
    chain_release();
    chain_wait();
    const int tid = threadIdx.x, T = blockDim.x, me = SMALL ? 0 : cl.block_rank(), n_cta = SMALL ? 1 : cl.num_blocks();
    const int gtid = me * T + tid, all = n_cta * T, cells = n_rows * width;
    const int32_t * tables = from.tables, * refs = from.refs;
    int32_t * held = to.refs;
    const bool out = !SMALL || blockIdx.x == 0;        // whether this CTA writes the result down
    int32_t * s_list = nullptr;                        // SMALL: the copies (src, dst, tokens), for this CTA's share of them
    if (tid == 0) sh.err = 0;
    for (int i = tid; i < n_rows; i += T) { s_raw[i] = from.lens[i]; s_par[i] = parent ? parent[i] : i; s_kept[i] = keep[i]; s_tot[i] = n_new[i]; }
    if (SMALL) {                                       // everything comes in at once
        int32_t * t = s_off + n_rows, * r = t + cells;
        held = r + n_pages; w.a = held + n_pages; w.b = w.a + n_pages; s_list = w.b + n_pages;
#pragma unroll 4
        for (int i = tid; i < cells; i += T) t[i] = tables[i];
#pragma unroll 4
        for (int i = tid; i < n_pages; i += T) r[i] = refs[i];
        tables = t; refs = r;
    }
    __syncthreads();
    // 1. requests checked, columns filled in; counts as they are, free pages by rank; pages that will be written announced
    for (int i = tid; i < n_rows; i += T) {
        const int p = s_par[i], k = s_kept[i], n = s_tot[i], len = s_raw[i];
        const bool ok = p >= 0 && p < n_rows && k >= 0 && n >= 0 && len >= 0 && (int64_t) k + n <= (int64_t) width * ps && len <= (int64_t) width * ps && k <= s_raw[p];
        if (!ok) sh.err = 1;
        const int full = k / ps, mod = k - full * ps;
        s_par[i] = ok ? p : i; s_old[i] = ok ? pg_ceil(len, ps) : 0; s_kept[i] = ok ? full + (mod != 0) : 0; s_tot[i] = ok ? pg_ceil(k + n, ps) : 0;
        s_len[i] = ok ? k + n : 0; s_mod[i] = ok && n > 0 ? mod : 0;
    }
    const int per = (n_pages + all - 1) / all, p0 = min(n_pages, gtid * per), p1 = min(n_pages, p0 + per);
    int my_free = 0;
    for (int p = p0; p < p1; p += PG_BATCH) {
        int r[PG_BATCH];
#pragma unroll
        for (int x = 0; x < PG_BATCH; ++x) r[x] = p + x < p1 ? refs[p + x] : 1;
#pragma unroll
        for (int x = 0; x < PG_BATCH; ++x) if (p + x < p1) { held[p + x] = r[x]; my_free += r[x] == 0; }
    }
    int cta_free;
    int free_before = pg_scan(my_free, sh.warp, &cta_free);            // (its barriers publish the columns)
    if (tid == 0) sh.n = cta_free;
    for (int i = gtid; i < n_rows; i += all) {
        const int s = s_mod[i] ? tables[s_par[i] * width + s_kept[i] - 1] : -1;
        if (s >= 0 && s < n_pages) { w.a[s] = 0x7fffffff; w.b[s] = 0; }
    }
    pg_sync<SMALL>(cl);
    // 2. old holders out, new ones in (what both have in the same column cancels); first writer and number of writers of a page.  Every entry
    // that is used has to be a page that is held (a free one would be given away as new); where one is not, `to` is made a copy of `from` in the end.
    // The counts are looked at one batch later, when they are there (64 x 5 rows of 259 pages: 20.7 us without, 22.0 at once, 21.7 so)
    int r[PG_BATCH];
#pragma unroll
    for (int x = 0; x < PG_BATCH; ++x) r[x] = 1;
    for (int c0 = gtid; c0 < cells; c0 += PG_BATCH * all) {
        int o[PG_BATCH], n[PG_BATCH];
#pragma unroll
        for (int x = 0; x < PG_BATCH; ++x) {
            const int c = c0 + x * all, i = (unsigned) c / (unsigned) width, j = c - i * width;
            const bool in = c < cells;
            o[x] = in && j < s_old[i] ? tables[c] : -1;
            n[x] = in && j < s_kept[i] ? tables[s_par[i] * width + j] : -1;
            if (in && j < s_old[i] && (o[x] < 0 || o[x] >= n_pages)) { sh.err = 1; o[x] = -1; }
        }
#pragma unroll
        for (int x = 0; x < PG_BATCH; ++x) {
            if (r[x] == 0) sh.err = 1;
            r[x] = o[x] >= 0 ? refs[o[x]] : 1;
        }
#pragma unroll
        for (int x = 0; x < PG_BATCH; ++x) if (o[x] != n[x]) {
            if (o[x] >= 0) atomicSub(&held[o[x]], 1);
            if (n[x] >= 0 && n[x] < n_pages) atomicAdd(&held[n[x]], 1);
        }
    }
    __syncthreads();                                    // s_page takes the place of s_old
    for (int i = tid; i < n_rows; i += T) {
        const int s = s_mod[i] ? tables[s_par[i] * width + s_kept[i] - 1] : -1;
        s_page[i] = s;
        if (i % n_cta == me && s >= 0 && s < n_pages) { atomicMin(&w.a[s], i); atomicAdd(&w.b[s], 1); }
    }
#pragma unroll
    for (int x = 0; x < PG_BATCH; ++x) if (r[x] == 0) sh.err = 1;
    int n_free, err;
    pg_across<SMALL>(cl, sh, &my_free, &n_free, &err);
    free_before += my_free;
    // 3. who copies, what is wanted (every CTA for itself)
    int wanted = 0, n_copy = 0;
    if (!err) {
        for (int i0 = 0; i0 < n_rows; i0 += T) {
            const int i = i0 + tid;
            int want = 0, copy = 0, s = -1;
            if (i < n_rows) {
                s = s_page[i];
                copy = s >= 0 && (pg_get<SMALL>(&w.a[s]) != i || pg_get<SMALL>(&held[s]) > pg_get<SMALL>(&w.b[s]));
                want = s_tot[i] - s_kept[i] + copy;
            }
            long long sum;                              // pages wanted (at most n_rows * (width + 1): below 2^31 by the host's check), copies from bit 40 on
            const long long at = pg_scan((long long) want | (long long) copy << 40, sh.warp2, &sum);
            const int before = wanted + (int) (at & 0x7fffffff);
            if (i < n_rows) s_off[i] = before | copy << 31;
            if (me == 0 && copy) {                      // destination: filled in below, when the free pages are known
                int32_t * l = (SMALL ? s_list : w.copies) + 3 * (n_copy + (int) (at >> 40));
                l[0] = s; l[1] = before; l[2] = s_mod[i];
            }
            wanted += (int) (sum & 0x7fffffff);
            n_copy += (int) (sum >> 40);
        }
    }
    const int missing = err ? -1 : max(wanted - n_free, 0);
    pg_sync<SMALL>(cl);                                 // all have read the counts and the writers: w.a becomes the list of free pages
    if (missing != 0) {
        if (!out) return;
        for (int p = gtid; p < n_pages; p += all) to.refs[p] = refs[p];
        for (int i = gtid; i < n_rows; i += all) to.lens[i] = from.lens[i];
        for (int c = gtid; c < cells; c += all) to.tables[c] = tables[c];
        if (gtid == 0) { status[0] = missing; status[1] = 0; w.head[0] = 0; }
        return;
    }
    for (int p = p0, f = free_before; p < p1 && f < wanted; p += PG_BATCH) {
        int r[PG_BATCH];
#pragma unroll
        for (int x = 0; x < PG_BATCH; ++x) r[x] = p + x < p1 ? refs[p + x] : 1;
#pragma unroll
        for (int x = 0; x < PG_BATCH; ++x) if (r[x] == 0 && f < wanted) { w.a[f++] = p + x; held[p + x] = 1; }
    }
    for (int i = gtid; i < n_rows; i += all) {
        if (out) to.lens[i] = s_len[i];
        if ((unsigned) s_off[i] >> 31) atomicSub(&held[s_page[i]], 1);
    }
    pg_sync<SMALL>(cl);
    // 4. the new tables
    for (int c0 = gtid; out && c0 < cells; c0 += PG_BATCH * all) {
        int t[PG_BATCH];
#pragma unroll
        for (int x = 0; x < PG_BATCH; ++x) {
            t[x] = -1;
            const int c = c0 + x * all, i = (unsigned) c / (unsigned) width, j = c - i * width;
            if (c < cells && j < s_tot[i]) {
                const int first = s_kept[i] - (int) ((unsigned) s_off[i] >> 31);
                t[x] = pg_get<SMALL>(j < first ? &tables[s_par[i] * width + j] : &w.a[(s_off[i] & 0x7fffffff) + j - first]);
            }
        }
#pragma unroll
        for (int x = 0; x < PG_BATCH; ++x) if (c0 + x * all < cells) to.tables[c0 + x * all] = t[x];
    }
    if (SMALL && out) for (int p = tid; p < n_pages; p += T) to.refs[p] = held[p];
    if (me == 0) {
        for (int c = tid; c < n_copy; c += T) {
            int32_t * l = (SMALL ? s_list : w.copies) + 3 * c;
            l[1] = pg_get<SMALL>(&w.a[l[1]]);
            if (SMALL && out) { w.copies[3 * c] = l[0]; w.copies[3 * c + 1] = l[1]; w.copies[3 * c + 2] = l[2]; }
        }
        if (tid == 0 && out) { status[0] = 0; status[1] = n_copy; w.head[0] = n_copy; }
    }
    if (SMALL && fused) {
        __syncthreads();
        pg_copy(pool, n_copy, blockIdx.x, gridDim.x, [&](int64_t c, int & src, int & dst, int & tokens) { src = s_list[3 * c]; dst = s_list[3 * c + 1]; tokens = s_list[3 * c + 2]; });
    }
}

template <bool SMALL>
__global__ void __launch_bounds__(PG_THREADS)
k_pages_compact(PgState from, PgState to, int n_rows, int width, int n_pages, int ps, int32_t * remap, int32_t * status, PgWork w,
                const __grid_constant__ b200_page_pool pool, bool fused) {
    cg::cluster_group cl = cg::this_cluster();
    __shared__ PgShared sh;
    __shared__ int s_low;
    extern __shared__ int32_t s_dyn[];
    chain_release();
    chain_wait();
    const int tid = threadIdx.x, T = blockDim.x, me = SMALL ? 0 : cl.block_rank(), n_cta = SMALL ? 1 : cl.num_blocks();
    const int gtid = me * T + tid, all = n_cta * T;
    const int cells = n_rows * width;
    const int32_t * tables = from.tables, * lens = from.lens, * refs = from.refs;
    int32_t * map = remap, * low_at = SMALL ? &s_low : &w.head[2];
    const bool out = !SMALL || blockIdx.x == 0;        // whether this CTA writes the result down
    if (tid == 0) sh.err = 0;
    if (SMALL) {
        int32_t * t = s_dyn, * l = t + cells, * r = l + n_rows;
        map = r + n_pages; w.a = map + n_pages; w.b = w.a + n_pages;
        for (int i = tid; i < n_rows; i += T) l[i] = lens[i];
#pragma unroll 4
        for (int i = tid; i < n_pages; i += T) r[i] = refs[i];
#pragma unroll 4
        for (int i = tid; i < cells; i += T) t[i] = tables[i];
        tables = t; lens = l; refs = r;
    }
    __syncthreads();
    const int per = (n_pages + all - 1) / all, p0 = min(n_pages, gtid * per), p1 = min(n_pages, p0 + per);
    int live = 0;
#pragma unroll 4
    for (int p = p0; p < p1; ++p) live += refs[p] != 0;
    int cta_live;
    int before = pg_scan(live, sh.warp, &cta_live);
    if (tid == 0) sh.n = cta_live;
    for (int i = gtid; i < n_rows; i += all) if (lens[i] < 0 || lens[i] > (int64_t) width * ps) sh.err = 1;
    for (int c0 = gtid; c0 < cells; c0 += PG_BATCH * all) {
        int t[PG_BATCH], n[PG_BATCH];
#pragma unroll
        for (int x = 0; x < PG_BATCH; ++x) {
            const int c = c0 + x * all, i = (unsigned) c / (unsigned) width;
            t[x] = c < cells && c - i * width < pg_ceil(max(lens[i], 0), ps) ? tables[c] : -2;       // -2: no page is looked for
        }
#pragma unroll
        for (int x = 0; x < PG_BATCH; ++x) n[x] = t[x] >= 0 && t[x] < n_pages ? refs[t[x]] : t[x] == -2;
#pragma unroll
        for (int x = 0; x < PG_BATCH; ++x) if (n[x] == 0) sh.err = 1;
    }
    int cta_before, n_live, err;
    pg_across<SMALL>(cl, sh, &cta_before, &n_live, &err);
    before += cta_before;
    // used pages by rank (w.a) and free pages by rank (w.b): the moves pair the tail of the first with the head of the second
    for (int p = p0, r = before; p < p1; ++p) {
        if (p == n_live) *low_at = r;                   // used pages below n_live
        if (refs[p] != 0) w.a[r++] = p;
        else              w.b[p - r] = p;
    }
    if (gtid == 0 && n_live == n_pages) *low_at = n_live;
    pg_sync<SMALL>(cl);
    const int low = pg_get<SMALL>(low_at), moves = err ? 0 : n_live - low;
    for (int p = p0, r = before; p < p1; ++p) {
        const int n = refs[p];
        int to_p = n != 0 ? p : -1, held = n;
        if (!err) {
            if (n != 0 && p >= n_live) to_p = pg_get<SMALL>(&w.b[r - low]);
            if (p >= n_live)   held = 0;
            else if (n == 0)   held = refs[pg_get<SMALL>(&w.a[low + p - r])];
        }
        if (out) to.refs[p] = held;
        map[p] = to_p;
        if (SMALL && out) remap[p] = to_p;
        r += n != 0;
    }
    for (int c = gtid; out && c < moves; c += all) { w.copies[3 * c] = pg_get<SMALL>(&w.a[low + c]); w.copies[3 * c + 1] = pg_get<SMALL>(&w.b[c]); w.copies[3 * c + 2] = ps; }
    if (gtid == 0 && out) { status[0] = err ? -1 : 0; status[1] = moves; w.head[0] = moves; }
    pg_sync<SMALL>(cl);
    for (int i = gtid; out && i < n_rows; i += all) to.lens[i] = lens[i];
    for (int c0 = gtid; out && c0 < cells; c0 += PG_BATCH * all) {
        int t[PG_BATCH];
#pragma unroll
        for (int x = 0; x < PG_BATCH; ++x) {
            const int c = c0 + x * all, i = (unsigned) c / (unsigned) width;
            t[x] = c < cells && (err || c - i * width < pg_ceil(lens[i], ps)) ? tables[c] : -1;
        }
        if (!err) {
#pragma unroll
            for (int x = 0; x < PG_BATCH; ++x) if (t[x] >= 0) t[x] = pg_get<SMALL>(&map[t[x]]);
        }
#pragma unroll
        for (int x = 0; x < PG_BATCH; ++x) if (c0 + x * all < cells) to.tables[c0 + x * all] = t[x];
    }
    if (SMALL && fused) pg_copy(pool, moves, blockIdx.x, gridDim.x, [&](int64_t c, int & src, int & dst, int & tokens) { src = w.a[low + c]; dst = w.b[c]; tokens = ps; });
}

// ---- host ----
// The list of copies is on the device, so its length is not known to the host: a grid of fixed size strides over it (18 000 pages of 64 KB:
// 211 us with 8 CTAs per SM in the grid, 193 with 64: 6.1 TB/s).
__global__ void __launch_bounds__(PG_COPY_THREADS)
k_pages_copy(b200_page_pool pool, const int32_t * head, const int32_t * copies, int most) {
    chain_release();
    chain_wait();
    pg_copy(pool, min(max(head[0], 0), most), blockIdx.x, gridDim.x, [&](int64_t c, int & src, int & dst, int & tokens) { src = copies[3 * c]; dst = copies[3 * c + 1]; tokens = copies[3 * c + 2]; });
}

bool b200_pool_ok(const b200_page_pool * p, bool data) {
    if (!p || p->n_pages < 1 || p->page_size < 1 || p->page_size > (1 << 20)) return false;
    if (!data) return true;
    if (!p->k || !p->v || (p->type != B200_TYPE_F16 && p->type != B200_TYPE_BF16) || (p->head_dim != 64 && p->head_dim != 128)) return false;
    if (p->n_layer < 1 || p->n_head_kv < 1 || p->n_head_kv > 1024) return false;
    if ((int64_t) p->page_size * p->n_head_kv * (p->head_dim / 8) > 0x7fffffff) return false;          // 16-byte vectors of a page
    const int64_t row = 2 * p->head_dim;
    const int64_t bits = (int64_t) (uintptr_t) p->k | (int64_t) (uintptr_t) p->v | p->nb_page | p->nb_tok | p->nb_head | (p->n_layer > 1 ? p->nb_layer : 0);
    if (bits % 16 || (p->n_head_kv > 1 && p->nb_head < row) || (p->page_size > 1 && p->nb_tok < row) || p->nb_page < row || p->nb_head < 0 || p->nb_tok < 0) return false;
    return true;
}

static int pg_launch_copy(const b200_page_pool * pool, const PgWork & w, int64_t max_copies, cudaStream_t st) {
    const int64_t tiles = ((int64_t) pool->page_size * pool->n_head_kv * pool->head_dim / 8 + PG_COPY_THREADS * PG_COPY_UNROLL - 1) / (PG_COPY_THREADS * PG_COPY_UNROLL);
    const int64_t items = max_copies * pool->n_layer * 2 * tiles;
    const unsigned grid = (unsigned) (items < 148 * 64 ? items : 148 * 64);
    const cudaError_t e = launch_chained(k_pages_copy, dim3(grid), dim3(PG_COPY_THREADS), 0, st, *pool, (const int32_t *) w.head, (const int32_t *) w.copies, (int) max_copies);
    if (e != cudaSuccess) return (int) e;
    B200_LAUNCHED();
    return 0;
}

// SMALL or cluster form of a kernel, by the size of the state; *fused: it makes the copies too (max_copies at most)
template <auto SMALL_KERNEL, auto LARGE_KERNEL, typename... Args>
static cudaError_t pg_launch(int64_t n_rows, int64_t width, int64_t n_pages, const b200_page_pool * pool, bool data, int64_t max_copies, bool * fused, cudaStream_t st, Args &&... args) {
    const int64_t words = pg_small_words(n_rows, width, n_pages);
    const bool fits = words * 4 <= PG_SMALL;
    *fused = fits && data && n_rows * width + n_pages <= PG_FUSED && n_rows <= PG_COPY_THREADS;
    cudaError_t e = fits ? allow_once<SMALL_KERNEL>(PG_SMALL) : allow_once<LARGE_KERNEL>(4 * PG_COLUMNS * PG_MAX_ROWS, true);
    if (e != cudaSuccess) return e;
    int64_t ctas = 1;
    if (*fused) {
        ctas = max_copies * pool->n_layer * 2 * (((int64_t) pool->page_size * pool->n_head_kv * pool->head_dim / 8 + PG_COPY_THREADS * PG_COPY_UNROLL - 1) / (PG_COPY_THREADS * PG_COPY_UNROLL));
        ctas = ctas < 1 ? 1 : ctas > 148 * 3 ? 148 * 3 : ctas;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned) (fits ? ctas : PG_CLUSTER));
    cfg.blockDim = dim3(*fused ? PG_COPY_THREADS : PG_THREADS);
    cfg.dynamicSmemBytes = (size_t) (fits ? words * 4 : 4 * PG_COLUMNS * (n_rows > 0 ? n_rows : 1));
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = fits ? 1 : PG_CLUSTER; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = b200_chained_launches() ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, fits ? SMALL_KERNEL : LARGE_KERNEL, std::forward<Args>(args)..., *pool, *fused);
}

// No output may overlap another one or an input: every CTA of a launch reads the inputs for itself, some of them when others already write.
struct PgSpan { const void * p; int64_t bytes; };
template <int OUT, int IN> static bool pg_apart(const PgSpan (&out)[OUT], const PgSpan (&in)[IN]) {
    auto meet = [](const PgSpan & a, const PgSpan & b) {
        return a.p && b.p && a.bytes > 0 && b.bytes > 0 && (uintptr_t) a.p < (uintptr_t) b.p + b.bytes && (uintptr_t) b.p < (uintptr_t) a.p + a.bytes;
    };
    for (int i = 0; i < OUT; ++i) {
        for (int j = 0; j < i; ++j) if (meet(out[i], out[j])) return false;
        for (int j = 0; j < IN; ++j) if (meet(out[i], in[j])) return false;
    }
    return true;
}

// what update and compact ask of their states
static bool pg_states_ok(const b200_page_state * from, const b200_page_state * to, int64_t n_pages, int64_t ps) {
    if (!from || !to || from->n_rows < 0 || from->n_rows > PG_MAX_ROWS || to->n_rows != from->n_rows || n_pages > PG_MAX_PAGES) return false;
    if (!from->refs || !to->refs || ((uintptr_t) from->refs | (uintptr_t) to->refs) % 4) return false;
    if (from->n_rows == 0) return true;
    if (from->table_stride < 1 || to->table_stride != from->table_stride || !from->tables || !to->tables || !from->lens || !to->lens) return false;
    const int64_t width = from->table_stride;
    if (((uintptr_t) from->tables | (uintptr_t) from->lens | (uintptr_t) to->tables | (uintptr_t) to->lens) % 4) return false;
    if (width >= (1ll << 30)) return false;
    return width * from->n_rows < (1ll << 30) && width * ps < (1ll << 31);
}

extern "C" int64_t b200_pages_workspace(int64_t n_rows, int64_t n_pages) {
    if (n_rows < 0 || n_rows > PG_MAX_ROWS || n_pages < 1 || n_pages > PG_MAX_PAGES) return 0;
    PgWork w;
    return pg_layout(&w, nullptr, n_rows, n_pages);
}

extern "C" int b200_pages_update(const b200_page_pool * pool, const b200_page_state * from, const b200_page_state * to, const int32_t * parent,
                                 const int32_t * keep, const int32_t * n_new, int32_t * status, void * workspace, int64_t workspace_bytes, void * stream) {
    const bool data = pool && (pool->k || pool->v);
    if (!b200_pool_ok(pool, data) || !pg_states_ok(from, to, pool->n_pages, pool->page_size) || !status) return B200_ERR_ARG;
    if ((from->n_rows && (!keep || !n_new)) || ((uintptr_t) parent | (uintptr_t) keep | (uintptr_t) n_new | (uintptr_t) status) % 4) return B200_ERR_ARG;
    if (!workspace || (uintptr_t) workspace % 16 || workspace_bytes < b200_pages_workspace(from->n_rows, pool->n_pages)) return B200_ERR_ARG;
    PgWork w;
    pg_layout(&w, workspace, from->n_rows, pool->n_pages);
    const PgState f = { from->tables, from->lens, from->refs }, t = { to->tables, to->lens, to->refs };
    const int width = from->n_rows ? (int) from->table_stride : 0;
    const int64_t rows = 4 * from->n_rows, cells = rows * width, pages = 4ll * pool->n_pages;
    if (!pg_apart({ { t.tables, cells }, { t.lens, rows }, { t.refs, pages }, { status, 8 }, { workspace, b200_pages_workspace(from->n_rows, pool->n_pages) } },
                  { { f.tables, cells }, { f.lens, rows }, { f.refs, pages }, { parent, rows }, { keep, rows }, { n_new, rows } })) return B200_ERR_ARG;
    const cudaStream_t st = as_stream(stream);
    bool fused;
    cudaError_t e = pg_launch<k_pages_update<true>, k_pages_update<false>>(from->n_rows, width, pool->n_pages, pool, data, from->n_rows, &fused, st, f, t, (int) from->n_rows, width, pool->n_pages, pool->page_size, parent, keep, n_new, status, w);
    if (e != cudaSuccess) return (int) e;
    B200_LAUNCHED();
    if (data && !fused && from->n_rows) return pg_launch_copy(pool, w, from->n_rows, st);
    return (int) cudaGetLastError();
}

extern "C" int b200_pages_compact(const b200_page_pool * pool, const b200_page_state * from, const b200_page_state * to, int32_t * remap,
                                  int32_t * status, void * workspace, int64_t workspace_bytes, void * stream) {
    const bool data = pool && (pool->k || pool->v);
    if (!b200_pool_ok(pool, data) || !pg_states_ok(from, to, pool->n_pages, pool->page_size) || !remap || !status || ((uintptr_t) remap | (uintptr_t) status) % 4) return B200_ERR_ARG;
    if (!workspace || (uintptr_t) workspace % 16 || workspace_bytes < b200_pages_workspace(from->n_rows, pool->n_pages)) return B200_ERR_ARG;
    PgWork w;
    pg_layout(&w, workspace, from->n_rows, pool->n_pages);
    const PgState f = { from->tables, from->lens, from->refs }, t = { to->tables, to->lens, to->refs };
    const int width = from->n_rows ? (int) from->table_stride : 0;
    const int64_t rows = 4 * from->n_rows, cells = rows * width, pages = 4ll * pool->n_pages;
    if (!pg_apart({ { t.tables, cells }, { t.lens, rows }, { t.refs, pages }, { remap, pages }, { status, 8 }, { workspace, b200_pages_workspace(from->n_rows, pool->n_pages) } },
                  { { f.tables, cells }, { f.lens, rows }, { f.refs, pages } })) return B200_ERR_ARG;
    const cudaStream_t st = as_stream(stream);
    bool fused;
    cudaError_t e = pg_launch<k_pages_compact<true>, k_pages_compact<false>>(from->n_rows, width, pool->n_pages, pool, data, pool->n_pages / 2 + 1, &fused, st, f, t, (int) from->n_rows, width, pool->n_pages, pool->page_size, remap, status, w);
    if (e != cudaSuccess) return (int) e;
    B200_LAUNCHED();
    if (data && !fused) return pg_launch_copy(pool, w, pool->n_pages / 2 + 1, st);
    return (int) cudaGetLastError();
}

extern "C" int b200_pages_copy(const b200_page_pool * pool, int64_t n_rows, const void * workspace, int64_t workspace_bytes, void * stream) {
    if (!b200_pool_ok(pool, true) || n_rows < 0 || n_rows > PG_MAX_ROWS || pool->n_pages > PG_MAX_PAGES) return B200_ERR_ARG;
    if (!workspace || (uintptr_t) workspace % 16 || workspace_bytes < b200_pages_workspace(n_rows, pool->n_pages)) return B200_ERR_ARG;
    PgWork w;
    pg_layout(&w, (void *) workspace, n_rows, pool->n_pages);
    const int64_t most = n_rows > pool->n_pages / 2 ? n_rows : pool->n_pages / 2 + 1;
    return pg_launch_copy(pool, w, most, as_stream(stream));
}
