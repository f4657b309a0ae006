// A paged key/value cache: who holds which page (fork, truncate, free, grow, compact) and the copies that follow from it.
// Counterpart in the reference: the cells of whisper_kv_cache (whisper_kv_cache_find_slot / _seq_cp / _seq_rm,
// src/whisper.cpp:1000-1200), which are host code over one dense cache.
#include "b200_common.cuh"
#include <cooperative_groups.h>
namespace cg = cooperative_groups;

// ---- tables and reference counts -----------------------------------------------------------------
// The steps depend on one another (counts -> who must copy -> which pages are taken), so all of them run in one launch.  A state that
// fits shared memory (SMALL) is loaded once and worked on there by one CTA; what bounds it is the latency of that load.  A larger one
// is the work of one cluster of CTAs on global memory: the hardware barrier of a cluster between the steps costs a fraction of a
// launch.  All results are integers and independent of the order of the atomics; ranks come from prefix sums.
#define PG_THREADS 1024
#define PG_CLUSTER 16
#define PG_MAX_ROWS 8192
#define PG_SMALL   (160 * 1024)   // bytes of shared memory that a small state may take
#define PG_HEADER  8              // workspace words before the lists: [0] copies, [1] tokens per whole page, [2] see k_pages_compact

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

// exclusive prefix sum over the block (values and total in 32 bits); s_warp: 33 words
__device__ __forceinline__ int pg_scan(int v, int * s_warp, int * total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int u = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += u; }
    __syncthreads();                                   // s_warp may still be read from the scan before
    if (lane == 31) s_warp[warp] = inc;
    __syncthreads();
    if (warp == 0) {
        const int x = s_warp[lane];
        int y = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int u = __shfl_up_sync(0xffffffffu, y, o); if (lane >= o) y += u; }
        s_warp[lane] = y - x;
        if (lane == 31) s_warp[32] = y;
    }
    __syncthreads();
    *total = s_warp[32];
    return s_warp[warp] + inc - v;
}

__device__ __forceinline__ int pg_ceil(int n, int ps) { return n / ps + (n % ps != 0); }

struct PgShared { int warp[33]; int n; int err; int pad; };

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
    else {
        const unsigned n = cl.num_blocks(), me = cl.block_rank();
        for (unsigned r = 0; r < n; ++r) {
            const PgShared * o = cl.map_shared_rank(&s, r);
            const int v = o->n;
            e |= o->err;
            if (r < me) b += v;
            t += v;
        }
    }
    *before = b; *all = t; *err = e;
}

// Loops over the cells of all tables and over a thread's run of pages load PG_BATCH values before they use the first: what they store may alias
// what they load as far as the compiler knows, and one value at a time costs a latency each (64 x 5 rows of 259 pages: 23 us).
#define PG_BATCH 4

// words of shared memory that a small state takes: tables, counts (as they are, and worked on), two lists of pages, columns of rows
#define PG_COLUMNS 7
static inline int64_t pg_small_words(int64_t n_rows, int64_t width, int64_t n_pages) { return n_rows * width + 4 * n_pages + PG_COLUMNS * n_rows; }

template <bool SMALL>
__global__ void __launch_bounds__(PG_THREADS)
k_pages_update(PgState from, PgState to, int n_rows, int width, int n_pages, int ps,
               const int32_t * parent, const int32_t * keep, const int32_t * n_new, int32_t * status, PgWork w) {
    cg::cluster_group cl = cg::this_cluster();
    __shared__ PgShared sh;
    extern __shared__ int32_t s_dyn[];
    // per row, in every CTA: its parent; pages it had, keeps, will have; its length; tokens in its last kept page if that will be written, else 0;
    // pages wanted by the rows before it (top bit: its last kept page is copied)
    int32_t * s_par = s_dyn, * s_old = s_par + n_rows, * s_kept = s_old + n_rows, * s_tot = s_kept + n_rows, * s_len = s_tot + n_rows, * s_mod = s_len + n_rows,
            * s_off = s_mod + n_rows;
    chain_release();
    chain_wait();
    const int tid = threadIdx.x, me = SMALL ? 0 : cl.block_rank(), n_cta = SMALL ? 1 : cl.num_blocks();
    const int gtid = me * PG_THREADS + tid, all = n_cta * PG_THREADS, cells = n_rows * width;
    const int32_t * tables = from.tables, * refs = from.refs;
    int32_t * held = to.refs;
    if (tid == 0) sh.err = 0;
    if (SMALL) {                                       // everything comes in at once
        int32_t * t = s_off + n_rows, * r = t + cells;
        held = r + n_pages; w.a = held + n_pages; w.b = w.a + n_pages;
#pragma unroll 4
        for (int i = tid; i < cells; i += PG_THREADS) t[i] = tables[i];
#pragma unroll 4
        for (int i = tid; i < n_pages; i += PG_THREADS) r[i] = refs[i];
        tables = t; refs = r;
    }
    __syncthreads();                                   // sh.err
    for (int i = tid; i < n_rows; i += PG_THREADS) {
        const int p = parent ? parent[i] : i, k = keep[i], n = n_new[i], len = from.lens[i];
        const bool in = p >= 0 && p < n_rows;
        const int have = in ? from.lens[p] : 0;
        const bool ok = in && k >= 0 && n >= 0 && len >= 0 && (int64_t) k + n <= (int64_t) width * ps && len <= (int64_t) width * ps && k <= have;
        if (!ok) sh.err = 1;
        s_par[i] = ok ? p : i; s_old[i] = ok ? pg_ceil(len, ps) : 0; s_kept[i] = ok ? pg_ceil(k, ps) : 0; s_tot[i] = ok ? pg_ceil(k + n, ps) : 0;
        s_len[i] = ok ? k + n : 0; s_mod[i] = ok && n > 0 ? k % ps : 0;
    }
    // 1. counts as they are, free pages by rank; pages that will be written announced; every entry that is read below has to be a page
    const int per = (n_pages + all - 1) / all, p0 = min(n_pages, gtid * per), p1 = min(n_pages, p0 + per);
    int my_free = 0;
    if (SMALL) __syncthreads();
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
    auto page_written = [&](int i) { return s_mod[i] ? tables[s_par[i] * width + s_kept[i] - 1] : -1; };
    for (int i = gtid; i < n_rows; i += all) {
        const int s = page_written(i);
        if (s >= 0 && s < n_pages) { w.a[s] = 0x7fffffff; w.b[s] = 0; }
    }
    for (int c0 = gtid; c0 < cells; c0 += PG_BATCH * all) {
        int t[PG_BATCH];
#pragma unroll
        for (int x = 0; x < PG_BATCH; ++x) t[x] = c0 + x * all < cells ? tables[c0 + x * all] : 0;
#pragma unroll
        for (int x = 0; x < PG_BATCH; ++x) {
            const int c = c0 + x * all, i = (unsigned) c / (unsigned) width;
            if ((t[x] < 0 || t[x] >= n_pages) && c - i * width < s_old[i]) sh.err = 1;
        }
    }
    int n_free, err;
    pg_across<SMALL>(cl, sh, &my_free, &n_free, &err);
    free_before += my_free;

    if (!err) {
        // 2. old holders out, new ones in (what both have in the same column cancels); first writer and number of writers of a page
        for (int c0 = gtid; c0 < cells; c0 += PG_BATCH * all) {
            int o[PG_BATCH], n[PG_BATCH];
#pragma unroll
            for (int x = 0; x < PG_BATCH; ++x) {
                const int c = c0 + x * all, i = (unsigned) c / (unsigned) width, j = c - i * width;
                const bool in = c < cells;
                o[x] = in && j < s_old[i] ? tables[c] : -1;
                n[x] = in && j < s_kept[i] ? tables[s_par[i] * width + j] : -1;
            }
#pragma unroll
            for (int x = 0; x < PG_BATCH; ++x) if (o[x] != n[x]) {
                if (o[x] >= 0) atomicSub(&held[o[x]], 1);
                if (n[x] >= 0) atomicAdd(&held[n[x]], 1);
            }
        }
        for (int i = gtid; i < n_rows; i += all) {
            const int s = page_written(i);
            if (s >= 0) { atomicMin(&w.a[s], i); atomicAdd(&w.b[s], 1); }
        }
    }
    pg_sync<SMALL>(cl);
    // 3. who copies, what is wanted (every CTA for itself)
    int wanted = 0, n_copy = 0;
    if (!err) {
        for (int i0 = 0; i0 < n_rows; i0 += PG_THREADS) {
            const int i = i0 + tid;
            int want = 0, copy = 0, s = -1;
            if (i < n_rows) {
                s = page_written(i);
                copy = s >= 0 && (pg_get<SMALL>(&w.a[s]) != i || pg_get<SMALL>(&held[s]) > pg_get<SMALL>(&w.b[s]));
                want = s_tot[i] - s_kept[i] + copy;
            }
            int sum;
            const int before = pg_scan(want, sh.warp, &sum);
            if (i < n_rows) s_off[i] = (wanted + before) | copy << 31;
            wanted += sum;                              // at most n_rows * (width + 1): checked to be below 2^31 by the host
            if (me == 0) {
                int copies;
                const int c_before = pg_scan(copy, sh.warp, &copies);
                if (copy) {                             // destination: filled in below, when the free pages are known
                    const int c = n_copy + c_before;
                    w.copies[3 * c] = s; w.copies[3 * c + 1] = wanted - sum + before; w.copies[3 * c + 2] = s_mod[i];
                }
                n_copy += copies;
            }
        }
    }
    const int missing = err ? -1 : max(wanted - n_free, 0);
    pg_sync<SMALL>(cl);                                 // all have read the counts and the writers: w.a becomes the list of free pages
    if (missing != 0) {
        for (int p = gtid; p < n_pages; p += all) to.refs[p] = refs[p];
        for (int i = gtid; i < n_rows; i += all) to.lens[i] = from.lens[i];
        for (int c = gtid; c < cells; c += all) to.tables[c] = tables[c];
        if (gtid == 0) { status[0] = missing; status[1] = 0; w.head[0] = 0; w.head[1] = ps; }
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
        to.lens[i] = s_len[i];
        if ((unsigned) s_off[i] >> 31) atomicSub(&held[page_written(i)], 1);
    }
    pg_sync<SMALL>(cl);
    // 4. the new tables
    for (int c0 = gtid; c0 < cells; c0 += PG_BATCH * all) {
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
    if (SMALL) for (int p = tid; p < n_pages; p += PG_THREADS) to.refs[p] = held[p];
    if (me == 0) {
        for (int c = tid; c < n_copy; c += PG_THREADS) w.copies[3 * c + 1] = pg_get<SMALL>(&w.a[w.copies[3 * c + 1]]);
        if (tid == 0) { status[0] = 0; status[1] = n_copy; w.head[0] = n_copy; w.head[1] = ps; }
    }
}

template <bool SMALL>
__global__ void __launch_bounds__(PG_THREADS)
k_pages_compact(PgState from, PgState to, int n_rows, int width, int n_pages, int ps, int32_t * remap, int32_t * status, PgWork w) {
    cg::cluster_group cl = cg::this_cluster();
    __shared__ PgShared sh;
    __shared__ int s_low;
    extern __shared__ int32_t s_dyn[];
    chain_release();
    chain_wait();
    const int tid = threadIdx.x, me = SMALL ? 0 : cl.block_rank(), n_cta = SMALL ? 1 : cl.num_blocks();
    const int gtid = me * PG_THREADS + tid, all = n_cta * PG_THREADS;
    const int cells = n_rows * width;
    const int32_t * tables = from.tables, * lens = from.lens, * refs = from.refs;
    int32_t * map = remap, * low_at = SMALL ? &s_low : &w.head[2];
    if (tid == 0) sh.err = 0;
    if (SMALL) {
        int32_t * t = s_dyn, * l = t + cells, * r = l + n_rows;
        map = r + n_pages; w.a = map + n_pages; w.b = w.a + n_pages;
        for (int i = tid; i < n_rows; i += PG_THREADS) l[i] = lens[i];
#pragma unroll 4
        for (int i = tid; i < n_pages; i += PG_THREADS) r[i] = refs[i];
#pragma unroll 4
        for (int i = tid; i < cells; i += PG_THREADS) t[i] = tables[i];
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
        to.refs[p] = held;
        map[p] = to_p;
        if (SMALL) remap[p] = to_p;
        r += n != 0;
    }
    for (int c = gtid; c < moves; c += all) { w.copies[3 * c] = pg_get<SMALL>(&w.a[low + c]); w.copies[3 * c + 1] = pg_get<SMALL>(&w.b[c]); w.copies[3 * c + 2] = ps; }
    if (gtid == 0) { status[0] = err ? -1 : 0; status[1] = moves; w.head[0] = moves; w.head[1] = ps; }
    pg_sync<SMALL>(cl);
    for (int i = gtid; i < n_rows; i += all) to.lens[i] = lens[i];
    for (int c0 = gtid; c0 < cells; c0 += PG_BATCH * all) {
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
}

// ---- copies --------------------------------------------------------------------------------------
// The list of copies is on the device, so its length is not known to the host: a fixed grid strides over
// (copy, layer, K or V, 16-byte vector).  Bound by memory for long lists: the bytes are read once and written once.
#define PG_COPY_THREADS 256
#define PG_COPY_UNROLL  4
__global__ void __launch_bounds__(PG_COPY_THREADS)
k_pages_copy(b200_page_pool pool, const int32_t * head, const int32_t * copies) {
    chain_release();
    chain_wait();
    const int n = head[0];
    const unsigned vec_head = pool.head_dim / 8, vec_tok = vec_head * pool.n_head_kv, vec_page = vec_tok * pool.page_size;
    const unsigned tiles = (vec_page + PG_COPY_THREADS * PG_COPY_UNROLL - 1) / (PG_COPY_THREADS * PG_COPY_UNROLL);
    const int64_t items = (int64_t) n * pool.n_layer * 2 * tiles;
    const int64_t row = pool.head_dim * 2;
    const bool toks = (pool.n_head_kv == 1 || pool.nb_head == row) && (pool.page_size == 1 || pool.nb_tok == row * pool.n_head_kv);
    const bool heads = (pool.page_size == 1 || pool.nb_tok == row) && (pool.n_head_kv == 1 || pool.nb_head == row * pool.page_size);
    for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
        int64_t r = it;
        const unsigned tile = (unsigned) (r % tiles); r /= tiles;
        const int kv = (int) (r & 1); r >>= 1;
        const int layer = (int) (r % pool.n_layer);
        const int64_t c = r / pool.n_layer;
        const int32_t src = copies[3 * c], dst = copies[3 * c + 1];
        const unsigned used = copies[3 * c + 2] * vec_tok;
        if (src < 0 || dst < 0 || src >= pool.n_pages || dst >= pool.n_pages || used > vec_page) continue;
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
                else { const unsigned per = copies[3 * c + 2] * vec_head; h = x / per; const unsigned y = x - h * per; tok = y / vec_head; i = y - tok * vec_head; }
                off[u] = tok * pool.nb_tok + h * pool.nb_head + i * 16;
                v[u] = *(const uint4 *) (base + src * pool.nb_page + off[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < PG_COPY_UNROLL; ++u) if (off[u] >= 0) *(uint4 *) (base + dst * pool.nb_page + off[u]) = v[u];
    }
}

bool b200_pool_ok(const b200_page_pool * p, bool data) {
    if (!p || p->n_pages < 1 || p->page_size < 1 || p->page_size > (1 << 20)) return false;
    if (!data) return true;
    if (!p->k || !p->v || (p->type != B200_TYPE_F16 && p->type != B200_TYPE_BF16) || (p->head_dim != 64 && p->head_dim != 128)) return false;
    if (p->n_layer < 1 || p->n_head_kv < 1 || p->n_head_kv > 1024) return false;
    const int64_t row = 2 * p->head_dim;
    const int64_t bits = (int64_t) (uintptr_t) p->k | (int64_t) (uintptr_t) p->v | p->nb_page | p->nb_tok | p->nb_head | (p->n_layer > 1 ? p->nb_layer : 0);
    if (bits % 16 || (p->n_head_kv > 1 && p->nb_head < row) || (p->page_size > 1 && p->nb_tok < row) || p->nb_page < row || p->nb_head < 0 || p->nb_tok < 0) return false;
    return true;
}

static int pg_launch_copy(const b200_page_pool * pool, const PgWork & w, int64_t max_copies, cudaStream_t st) {
    const int64_t tiles = ((int64_t) pool->page_size * pool->n_head_kv * pool->head_dim / 8 + PG_COPY_THREADS * PG_COPY_UNROLL - 1) / (PG_COPY_THREADS * PG_COPY_UNROLL);
    const int64_t items = max_copies * pool->n_layer * 2 * tiles;
    const unsigned grid = (unsigned) (items < 148 * 8 ? items : 148 * 8);
    const cudaError_t e = launch_chained(k_pages_copy, dim3(grid), dim3(PG_COPY_THREADS), 0, st, *pool, (const int32_t *) w.head, (const int32_t *) w.copies);
    if (e != cudaSuccess) return (int) e;
    B200_LAUNCHED();
    return 0;
}

// SMALL or cluster form of a kernel, by the size of the state
template <typename... KArgs, typename... Args>
static cudaError_t pg_launch(void (*small)(KArgs...), void (*large)(KArgs...), int64_t n_rows, int64_t width, int64_t n_pages, cudaStream_t st, Args &&... args) {
    const int64_t words = pg_small_words(n_rows, width, n_pages);
    const bool fits = words * 4 <= PG_SMALL;
    auto kernel = fits ? small : large;
    const size_t smem = fits ? words * 4 : 4 * PG_COLUMNS * (n_rows > 0 ? n_rows : 1);
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, fits ? PG_SMALL : 4 * PG_COLUMNS * PG_MAX_ROWS);
    if (e == cudaSuccess && !fits) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    const unsigned n = fits ? 1 : PG_CLUSTER;
    cfg.gridDim = dim3(n); cfg.blockDim = dim3(PG_THREADS); cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = n; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = b200_chained_launches() ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

// what update and compact ask of their states
static bool pg_states_ok(const b200_page_state * from, const b200_page_state * to, int64_t n_pages, int64_t ps) {
    if (!from || !to || from->n_rows < 0 || from->n_rows > PG_MAX_ROWS || to->n_rows != from->n_rows) return false;
    if (from->n_rows == 0) return from->refs && to->refs && from->refs != to->refs;
    if (from->table_stride < 1 || to->table_stride != from->table_stride || !from->tables || !to->tables || !from->lens || !to->lens || !from->refs || !to->refs) return false;
    const int64_t width = from->table_stride;
    if (width >= (1ll << 30)) return false;
    if (width * from->n_rows >= (1ll << 30) || width * ps >= (1ll << 31)) return false;
    auto apart = [](const void * a, int64_t na, const void * b, int64_t nb) { return (const char *) a + na <= (const char *) b || (const char *) b + nb <= (const char *) a; };
    return apart(from->tables, 4 * from->table_stride * from->n_rows, to->tables, 4 * to->table_stride * to->n_rows) &&
           apart(from->lens, 4 * from->n_rows, to->lens, 4 * to->n_rows) && apart(from->refs, 4 * n_pages, to->refs, 4 * n_pages);
}

extern "C" int64_t b200_pages_workspace(int64_t n_rows, int64_t n_pages) {
    if (n_rows < 0 || n_rows > PG_MAX_ROWS || n_pages < 1 || n_pages > 0x7fffffff) return 0;
    PgWork w;
    return pg_layout(&w, nullptr, n_rows, n_pages);
}

extern "C" int b200_pages_update(const b200_page_pool * pool, const b200_page_state * from, const b200_page_state * to, const int32_t * parent,
                                 const int32_t * keep, const int32_t * n_new, int32_t * status, void * workspace, int64_t workspace_bytes, void * stream) {
    const bool data = pool && (pool->k || pool->v);
    if (!b200_pool_ok(pool, data) || !pg_states_ok(from, to, pool->n_pages, pool->page_size) || !status) return B200_ERR_ARG;
    if (from->n_rows && (!keep || !n_new)) return B200_ERR_ARG;
    if (!workspace || (uintptr_t) workspace % 16 || workspace_bytes < b200_pages_workspace(from->n_rows, pool->n_pages)) return B200_ERR_ARG;
    PgWork w;
    pg_layout(&w, workspace, from->n_rows, pool->n_pages);
    const PgState f = { from->tables, from->lens, from->refs }, t = { to->tables, to->lens, to->refs };
    const int width = from->n_rows ? (int) from->table_stride : 0;
    const cudaStream_t st = as_stream(stream);
    cudaError_t e = pg_launch(k_pages_update<true>, k_pages_update<false>, from->n_rows, width, pool->n_pages, st, f, t, (int) from->n_rows, width, pool->n_pages, pool->page_size, parent, keep, n_new, status, w);
    if (e != cudaSuccess) return (int) e;
    B200_LAUNCHED();
    if (data && from->n_rows) return pg_launch_copy(pool, w, from->n_rows, st);
    return (int) cudaGetLastError();
}

extern "C" int b200_pages_compact(const b200_page_pool * pool, const b200_page_state * from, const b200_page_state * to, int32_t * remap,
                                  int32_t * status, void * workspace, int64_t workspace_bytes, void * stream) {
    const bool data = pool && (pool->k || pool->v);
    if (!b200_pool_ok(pool, data) || !pg_states_ok(from, to, pool->n_pages, pool->page_size) || !remap || !status) return B200_ERR_ARG;
    if (!workspace || (uintptr_t) workspace % 16 || workspace_bytes < b200_pages_workspace(from->n_rows, pool->n_pages)) return B200_ERR_ARG;
    PgWork w;
    pg_layout(&w, workspace, from->n_rows, pool->n_pages);
    const PgState f = { from->tables, from->lens, from->refs }, t = { to->tables, to->lens, to->refs };
    const int width = from->n_rows ? (int) from->table_stride : 0;
    const cudaStream_t st = as_stream(stream);
    cudaError_t e = pg_launch(k_pages_compact<true>, k_pages_compact<false>, from->n_rows, width, pool->n_pages, st, f, t, (int) from->n_rows, width, pool->n_pages, pool->page_size, remap, status, w);
    if (e != cudaSuccess) return (int) e;
    B200_LAUNCHED();
    if (data) return pg_launch_copy(pool, w, pool->n_pages / 2 + 1, st);
    return (int) cudaGetLastError();
}

extern "C" int b200_pages_copy(const b200_page_pool * pool, int64_t n_rows, const void * workspace, int64_t workspace_bytes, void * stream) {
    if (!b200_pool_ok(pool, true) || n_rows < 0 || n_rows > PG_MAX_ROWS) return B200_ERR_ARG;
    if (!workspace || (uintptr_t) workspace % 16 || workspace_bytes < b200_pages_workspace(n_rows, pool->n_pages)) return B200_ERR_ARG;
    PgWork w;
    pg_layout(&w, (void *) workspace, n_rows, pool->n_pages);
    const int64_t most = n_rows > pool->n_pages / 2 ? n_rows : pool->n_pages / 2 + 1;
    return pg_launch_copy(pool, w, most, as_stream(stream));
}
