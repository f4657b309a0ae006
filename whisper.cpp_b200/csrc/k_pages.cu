// A paged key/value cache: who holds which page (fork, truncate, free, grow, compact) and the copies that follow from it.
// Counterpart in the reference: the cells of whisper_kv_cache (whisper_kv_cache_find_slot / _seq_cp / _seq_rm,
// src/whisper.cpp:1000-1200), which are host code over one dense cache.
#include "b200_common.cuh"
#include <cooperative_groups.h>
namespace cg = cooperative_groups;

// ---- tables and reference counts -----------------------------------------------------------------
// One cluster of CTAs does all of it: the steps depend on one another (counts -> who must copy -> which pages are taken), and
// the hardware barrier of a cluster between them costs a fraction of a launch.  A small problem runs in one CTA.  What is
// bound here is latency: the tables of 320 rows are 330 KB, a third of a microsecond of memory time.  All results are
// integers and independent of the order of the atomics; ranks come from prefix sums.
#define PG_THREADS 1024
#define PG_CLUSTER 8
#define PG_MAX_ROWS 8192
#define PG_HEADER  8           // workspace words before the lists: [0] copies, [1] tokens per whole page, rest unused

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

// this CTA's contribution -> sum over the CTAs before it, and over all (reads the others' shared memory: barriers around it)
__device__ __forceinline__ void pg_across(cg::cluster_group & cl, PgShared & s, int * before, int * all, int * err) {
    cl.sync();
    int b = 0, t = 0, e = 0;
    const unsigned n = cl.num_blocks(), me = cl.block_rank();
    for (unsigned r = 0; r < n; ++r) {
        const PgShared * o = cl.map_shared_rank(&s, r);
        const int v = o->n;
        e |= o->err;
        if (r < me) b += v;
        t += v;
    }
    *before = b; *all = t; *err = e;
}

__global__ void __launch_bounds__(PG_THREADS)
k_pages_update(PgState from, PgState to, int n_rows, int width, int n_pages, int ps,
               const int32_t * parent, const int32_t * keep, const int32_t * n_new, int32_t * status, PgWork w) {
    cg::cluster_group cl = cg::this_cluster();
    __shared__ PgShared sh;
    extern __shared__ int32_t s_off[];                 // per row: pages wanted by the rows before it, top bit: its last page is copied
    chain_release();
    chain_wait();
    const int tid = threadIdx.x, me = cl.block_rank(), n_cta = cl.num_blocks();
    const int gtid = me * PG_THREADS + tid, all = n_cta * PG_THREADS;
    const int lane = tid & 31, gwarp = gtid >> 5, n_gwarp = all >> 5;
    if (tid == 0) sh.err = 0;
    __syncthreads();

    // 1. counts as they are; requests checked; pages that will be written announced
    const int per = (n_pages + all - 1) / all, p0 = min(n_pages, gtid * per), p1 = min(n_pages, p0 + per);
    int my_free = 0;
    for (int p = p0; p < p1; ++p) { const int r = from.refs[p]; to.refs[p] = r; my_free += r == 0; }
    int cta_free;
    int free_before = pg_scan(my_free, sh.warp, &cta_free);
    if (tid == 0) sh.n = cta_free;
    auto row_src = [&](int i) { const int p = parent ? parent[i] : i; return p; };
    auto page_written = [&](int i, int p) { const int k = keep[i]; return k % ps != 0 && n_new[i] > 0 ? from.tables[p * (int64_t) width + k / ps] : -1; };
    for (int i = gtid; i < n_rows; i += all) {
        const int p = row_src(i), k = keep[i], n = n_new[i], len = from.lens[i];
        bool ok = p >= 0 && p < n_rows && k >= 0 && n >= 0 && len >= 0 && (int64_t) k + n <= (int64_t) width * ps && len <= (int64_t) width * ps;
        ok = ok && k <= from.lens[p];
        if (!ok) { sh.err = 1; continue; }
        const int s = page_written(i, p);
        if (s >= 0 && s < n_pages) { w.a[s] = 0x7fffffff; w.b[s] = 0; }
    }
    // every table entry that is read below has to be a page
    for (int i = gwarp; i < n_rows; i += n_gwarp) {
        const int used = min(pg_ceil(max(from.lens[i], 0), ps), width);
        for (int j = lane; j < used; j += 32) { const int t = from.tables[i * (int64_t) width + j]; if (t < 0 || t >= n_pages) sh.err = 1; }
    }
    int n_free, err;
    pg_across(cl, sh, &my_free, &n_free, &err);
    free_before += my_free;

    if (!err) {
        // 2. old holders out, new ones in (what both have in the same column cancels); first writer and number of writers of a page
        for (int i = gwarp; i < n_rows; i += n_gwarp) {
            const int p = row_src(i), old_n = pg_ceil(from.lens[i], ps), new_n = pg_ceil(keep[i], ps);
            for (int j = lane; j < max(old_n, new_n); j += 32) {
                const int o = j < old_n ? from.tables[i * (int64_t) width + j] : -1, n = j < new_n ? from.tables[p * (int64_t) width + j] : -1;
                if (o != n) {
                    if (o >= 0) atomicSub(&to.refs[o], 1);
                    if (n >= 0) atomicAdd(&to.refs[n], 1);
                }
            }
            if (lane == 0) {
                const int s = page_written(i, p);
                if (s >= 0) { atomicMin(&w.a[s], i); atomicAdd(&w.b[s], 1); }
            }
        }
    }
    cl.sync();
    // 3. who copies, what is wanted (every CTA for itself)
    int wanted = 0, n_copy = 0;
    if (!err) {
        for (int i0 = 0; i0 < n_rows; i0 += PG_THREADS) {
            const int i = i0 + tid;
            int want = 0, copy = 0;
            if (i < n_rows) {
                const int s = page_written(i, row_src(i));
                copy = s >= 0 && (__ldcg(&w.a[s]) != i || __ldcg(&to.refs[s]) > __ldcg(&w.b[s]));
                want = pg_ceil(keep[i] + n_new[i], ps) - pg_ceil(keep[i], ps) + copy;
            }
            int sum;
            const int before = pg_scan(want, sh.warp, &sum);
            if (i < n_rows) s_off[i] = (wanted + before) | copy << 31;
            wanted += sum;                              // at most n_rows * width: checked to be below 2^31 by the host
            if (me == 0) {
                int copies;
                const int c_before = pg_scan(copy, sh.warp, &copies);
                if (copy) {                             // destination: filled in below, when the free pages are known
                    const int s = page_written(i, row_src(i)), c = n_copy + c_before;
                    w.copies[3 * c] = s; w.copies[3 * c + 1] = wanted - sum + before; w.copies[3 * c + 2] = keep[i] % ps;
                }
                n_copy += copies;
            }
        }
    }
    const int missing = err ? -1 : max(wanted - n_free, 0);
    cl.sync();                                          // all have read the counts and the writers: w.a becomes the list of free pages
    if (missing != 0) {
        for (int p = gtid; p < n_pages; p += all) to.refs[p] = from.refs[p];
        for (int i = gtid; i < n_rows; i += all) to.lens[i] = from.lens[i];
        for (int i = gwarp; i < n_rows; i += n_gwarp)
            for (int j = lane; j < width; j += 32) to.tables[i * (int64_t) width + j] = from.tables[i * (int64_t) width + j];
        if (gtid == 0) { status[0] = missing; status[1] = 0; w.head[0] = 0; w.head[1] = ps; }
        return;
    }
    for (int p = p0, r = free_before; p < p1 && r < wanted; ++p)
        if (from.refs[p] == 0) { w.a[r++] = p; to.refs[p] = 1; }
    cl.sync();
    // 4. the new tables
    for (int i = gwarp; i < n_rows; i += n_gwarp) {
        const int p = row_src(i), k = keep[i], o = s_off[i] & 0x7fffffff, copy = (unsigned) s_off[i] >> 31;
        const int first = pg_ceil(k, ps) - copy, total = pg_ceil(k + n_new[i], ps);
        for (int j = lane; j < width; j += 32) {
            int t = -1;
            if (j < first)      t = from.tables[p * (int64_t) width + j];
            else if (j < total) t = __ldcg(&w.a[o + j - first]);
            to.tables[i * (int64_t) width + j] = t;
        }
        if (lane == 0) {
            to.lens[i] = k + n_new[i];
            if (copy) atomicSub(&to.refs[from.tables[p * (int64_t) width + first]], 1);
        }
    }
    if (me == 0) {
        for (int c = tid; c < n_copy; c += PG_THREADS) w.copies[3 * c + 1] = __ldcg(&w.a[w.copies[3 * c + 1]]);
        if (tid == 0) { status[0] = 0; status[1] = n_copy; w.head[0] = n_copy; w.head[1] = ps; }
    }
}

__global__ void __launch_bounds__(PG_THREADS)
k_pages_compact(PgState from, PgState to, int n_rows, int width, int n_pages, int ps,
                int32_t * remap, int32_t * status, PgWork w) {
    cg::cluster_group cl = cg::this_cluster();
    __shared__ PgShared sh;
    chain_release();
    chain_wait();
    const int tid = threadIdx.x, me = cl.block_rank(), n_cta = cl.num_blocks();
    const int gtid = me * PG_THREADS + tid, all = n_cta * PG_THREADS;
    const int lane = tid & 31, gwarp = gtid >> 5, n_gwarp = all >> 5;
    if (tid == 0) sh.err = 0;
    __syncthreads();
    const int per = (n_pages + all - 1) / all, p0 = min(n_pages, gtid * per), p1 = min(n_pages, p0 + per);
    int live = 0;
    for (int p = p0; p < p1; ++p) live += from.refs[p] != 0;
    int cta_live;
    int before = pg_scan(live, sh.warp, &cta_live);
    if (tid == 0) sh.n = cta_live;
    for (int i = gwarp; i < n_rows; i += n_gwarp) {
        const int len = from.lens[i];
        if (len < 0 || len > (int64_t) width * ps) { sh.err = 1; continue; }
        for (int j = lane; j < pg_ceil(len, ps); j += 32) {
            const int t = from.tables[i * (int64_t) width + j];
            if (t < 0 || t >= n_pages || from.refs[t] == 0) sh.err = 1;
        }
    }
    int cta_before, n_live, err;
    pg_across(cl, sh, &cta_before, &n_live, &err);
    before += cta_before;
    // used pages by rank (w.a) and free pages by rank (w.b): the moves pair the tail of the first with the head of the second
    for (int p = p0, r = before; p < p1; ++p) {
        if (p == n_live) w.head[2] = r;                 // used pages below n_live
        if (from.refs[p] != 0) w.a[r++] = p;
        else                   w.b[p - r] = p;
    }
    if (gtid == 0 && n_live == n_pages) w.head[2] = n_live;
    cl.sync();
    const int low = __ldcg(&w.head[2]), moves = err ? 0 : n_live - low;
    for (int p = p0, r = before; p < p1; ++p) {
        const int refs = from.refs[p];
        int to_p = refs != 0 ? p : -1;
        if (!err) {
            if (refs != 0 && p >= n_live) to_p = __ldcg(&w.b[r - low]);
            if (p >= n_live)        to.refs[p] = 0;
            else if (refs != 0)     to.refs[p] = refs;
            else                    to.refs[p] = from.refs[__ldcg(&w.a[low + p - r])];
        } else to.refs[p] = refs;
        remap[p] = to_p;
        r += refs != 0;
    }
    for (int c = gtid; c < moves; c += all) { w.copies[3 * c] = __ldcg(&w.a[low + c]); w.copies[3 * c + 1] = __ldcg(&w.b[c]); w.copies[3 * c + 2] = ps; }
    if (gtid == 0) { status[0] = err ? -1 : 0; status[1] = moves; w.head[0] = moves; w.head[1] = ps; }
    cl.sync();
    for (int i = gtid; i < n_rows; i += all) to.lens[i] = from.lens[i];
    for (int i = gwarp; i < n_rows; i += n_gwarp) {
        const int used = err ? width : pg_ceil(from.lens[i], ps);
        for (int j = lane; j < width; j += 32) {
            int t = j < used ? from.tables[i * (int64_t) width + j] : -1;
            if (!err && j < used) t = __ldcg(&remap[t]);
            to.tables[i * (int64_t) width + j] = t;
        }
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
        uint4 v[PG_COPY_UNROLL];
        int64_t off[PG_COPY_UNROLL];
#pragma unroll
        for (int u = 0; u < PG_COPY_UNROLL; ++u) {
            const unsigned x = (tile * PG_COPY_UNROLL + u) * PG_COPY_THREADS + threadIdx.x;
            off[u] = -1;
            if (x < used) {
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

template <typename... KArgs, typename... Args>
static cudaError_t pg_launch(void (*kernel)(KArgs...), int64_t work, size_t smem, cudaStream_t st, Args &&... args) {
    cudaLaunchConfig_t cfg = {};
    const unsigned n = work <= 16 * PG_THREADS ? 1 : PG_CLUSTER;
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
    cudaError_t e = pg_launch(k_pages_update, from->n_rows * width + pool->n_pages, 4 * (size_t) from->n_rows, st, f, t, (int) from->n_rows, width, pool->n_pages, pool->page_size, parent, keep, n_new, status, w);
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
    cudaError_t e = pg_launch(k_pages_compact, from->n_rows * width + pool->n_pages, 0, st, f, t, (int) from->n_rows, width, pool->n_pages, pool->page_size, remap, status, w);
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
