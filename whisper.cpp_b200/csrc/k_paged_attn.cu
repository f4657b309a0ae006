// Attention of a chunk of new tokens over a paged key/value cache, single tokens included, and the store that precedes it.
// The reference has one dense cache per state (whisper_kv_cache, src/whisper.cpp:1000-1200) and decodes through
// ggml_compute_forward_flash_attn_ext_f16 (ggml/src/ggml-cpu/ops.cpp:6638-6851); this operator is defined by its formula
// (include/b200_whisper.h), with 32-bit scores, weights' sums and accumulators.
#include "b200_common.cuh"
#include <cuda_bf16.h>

bool b200_pool_ok(const b200_page_pool * p, bool data);    // k_pages.cu

struct PaArgs {
    const char * q; int64_t nb_q_tok, nb_q_head;
    char * dst; int64_t nb_dst_tok, nb_dst_head;
    const char * k; const char * v; int64_t nb_page, nb_tok, nb_head;
    const int32_t * tables; int64_t table_stride; const int32_t * lens; const int32_t * q_start;
    float * lse;
    float * part;                   // [split][n_tok * n_head] x (head_dim + 2): sums, maximum, sum of weights
    int64_t n_tok, max_len;
    int n_pages, page_size, n_head, n_head_kv, group, max_new, causal, n_split, chunk;
    float scale_log2;               // scale * log2(e): weights are powers of two
};

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

// ---- store ---------------------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ uint4 pa_pack8(const float * x);
template <> __device__ __forceinline__ uint4 pa_pack8<__half>(const float * x) {
    union { uint4 q; __half2 h[4]; } u;
#pragma unroll
    for (int i = 0; i < 4; ++i) u.h[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    return u.q;
}
template <> __device__ __forceinline__ uint4 pa_pack8<__nv_bfloat16>(const float * x) {
    union { uint4 q; __nv_bfloat162 h[4]; } u;
#pragma unroll
    for (int i = 0; i < 4; ++i) u.h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    return u.q;
}
template <typename T> __device__ __forceinline__ void pa_unpack8(uint4 q, float * x);
template <> __device__ __forceinline__ void pa_unpack8<__half>(uint4 q, float * x) {
    union { uint4 q; __half2 h[4]; } u; u.q = q;
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 f = __half22float2(u.h[i]); x[2 * i] = f.x; x[2 * i + 1] = f.y; }
}
template <> __device__ __forceinline__ void pa_unpack8<__nv_bfloat16>(uint4 q, float * x) {
    const uint32_t w[4] = { q.x, q.y, q.z, q.w };
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}

struct PaNew { const char * k; const char * v; int64_t nb_tok, nb_head; };

// one thread per 8 values; f32 is rounded to the pool's type (to nearest even: the cache's precision), 16-bit values are copied
template <typename KV, bool F32>
__global__ void __launch_bounds__(256)
k_paged_store(PaArgs a, PaNew x, int vec_head) {
    chain_release();
    chain_wait();
    const PaSeq s = pa_seq(a, blockIdx.y);
    const int per_tok = 2 * a.n_head_kv * vec_head;
    for (int64_t i = (int64_t) blockIdx.x * 256 + threadIdx.x; i < (int64_t) s.n_new * per_tok; i += (int64_t) gridDim.x * 256) {
        const int t = (int) (i / per_tok), r = (int) (i - (int64_t) t * per_tok), c = r % vec_head, h = r / vec_head % a.n_head_kv;
        const bool v = r >= per_tok / 2;
        const int pos = s.len - s.n_new + t;
        if (pos < 0) continue;
        const int page = a.tables[blockIdx.y * a.table_stride + pos / a.page_size];
        if (page < 0 || page >= a.n_pages) continue;
        const char * src = (v ? x.v : x.k) + (s.tok0 + t) * x.nb_tok + h * x.nb_head;
        uint4 q;
        if (F32) {
            float f[8];
            *(float4 *) f = ((const float4 *) src)[2 * c];
            *(float4 *) (f + 4) = ((const float4 *) src)[2 * c + 1];
            q = pa_pack8<KV>(f);
        } else q = ((const uint4 *) src)[c];
        *(uint4 *) ((char *) (v ? a.v : a.k) + page * a.nb_page + (pos % a.page_size) * a.nb_tok + h * a.nb_head + c * 16) = q;
    }
}

// ---- attention, one key per lane -----------------------------------------------------------------
// A CTA takes 8 rows (a row = one query token of one query head; rows of a key/value head are numbered token * group + head in
// group) of one sequence and key/value head, over one split of the keys; its four warps take every fourth block of 32 keys.
// Scores: a lane owns a key, the queries come from shared memory.  Products with V: a lane owns head_dim / 32 dimensions.
// Running maximum and sum per row; the warps, then the splits, are joined at the end.
#define PA_ROWS 8
template <typename Q, typename KV, int D>
__global__ void __launch_bounds__(128)
k_paged_attn(PaArgs a) {
    chain_release();
    chain_wait();
    constexpr int DL = D / 32;
    __shared__ float s_q[PA_ROWS][D];
    __shared__ float s_p[4][PA_ROWS][32];
    __shared__ float s_m[4][PA_ROWS], s_l[4][PA_ROWS];
    __shared__ float s_o[4][PA_ROWS][D];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int seq = blockIdx.z / a.n_split, split = blockIdx.z % a.n_split, kvh = blockIdx.y, row0 = blockIdx.x * PA_ROWS;
    const PaSeq s = pa_seq(a, seq);
    const int n_rows = s.n_new * a.group;
    if (row0 >= n_rows) return;
    const int last_t = (min(row0 + PA_ROWS, n_rows) - 1) / a.group;
    const int reach = a.causal ? min(s.len, max(s.len - s.n_new + last_t + 1, 0)) : s.len;      // keys that any row of the tile sees
    const int k0 = split * a.chunk, k1 = min(reach, k0 + a.chunk);
    if (k0 >= k1 && !(split == 0)) return;               // an empty split: the join does not read it
    for (int i = tid; i < PA_ROWS * D; i += 128) {
        const int r = row0 + i / D, t = r / a.group, h = kvh * a.group + r % a.group;
        s_q[i / D][i % D] = r < n_rows ? (float) ((const Q *) (a.q + (s.tok0 + t) * a.nb_q_tok + h * a.nb_q_head))[i % D] * a.scale_log2 : 0.0f;
    }
    int last[PA_ROWS];                                   // last key of every row
#pragma unroll
    for (int r = 0; r < PA_ROWS; ++r) last[r] = row0 + r >= n_rows ? -1 : a.causal ? s.len - s.n_new + (row0 + r) / a.group : s.len - 1;
    __syncthreads();
    float m[PA_ROWS], l[PA_ROWS], o[PA_ROWS][DL];
#pragma unroll
    for (int r = 0; r < PA_ROWS; ++r) { m[r] = -INFINITY; l[r] = 0.0f; for (int i = 0; i < DL; ++i) o[r][i] = 0.0f; }
    const int32_t * table = a.tables + seq * a.table_stride;
    for (int kb = k0 + warp * 32; kb < k1; kb += 128) {
        const int key = kb + lane;
        int64_t at = -1;
        if (key < k1) {
            const int page = table[key / a.page_size];
            if (page >= 0 && page < a.n_pages) at = page * a.nb_page + (key % a.page_size) * a.nb_tok + kvh * a.nb_head;
        }
        float sc[PA_ROWS] = {};
        if (at >= 0) {
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
                float kx[8];
                pa_unpack8<KV>(*(const uint4 *) (a.k + at + c * 16), kx);
#pragma unroll
                for (int r = 0; r < PA_ROWS; ++r)
#pragma unroll
                    for (int i = 0; i < 8; ++i) sc[r] = fmaf(s_q[r][c * 8 + i], kx[i], sc[r]);
            }
        }
#pragma unroll
        for (int r = 0; r < PA_ROWS; ++r) {
            const float x = key < k1 && key <= last[r] ? sc[r] : -INFINITY;
            float mx = x;
#pragma unroll
            for (int of = 16; of > 0; of >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, of));
            const float m1 = fmaxf(m[r], mx), base = m1 == -INFINITY ? 0.0f : m1;
            const float f = exp2f(m[r] - base), p = exp2f(x - base);
            l[r] = l[r] * f + p;
            m[r] = m1;
#pragma unroll
            for (int i = 0; i < DL; ++i) o[r][i] *= f;
            s_p[warp][r][lane] = p;
        }
        __syncwarp();
        const int n = min(32, k1 - kb);
        for (int j = 0; j < n; ++j) {
            const int64_t vat = __shfl_sync(0xffffffffu, at, j);
            if (vat < 0) continue;
            float vx[DL];
#pragma unroll
            for (int i = 0; i < DL; ++i) vx[i] = (float) ((const KV *) (a.v + vat))[lane * DL + i];
#pragma unroll
            for (int r = 0; r < PA_ROWS; ++r) {
                if (kb + j > last[r]) continue;            // not 0 * v: v may be infinite or NaN where the row does not look
                const float p = s_p[warp][r][j];
#pragma unroll
                for (int i = 0; i < DL; ++i) o[r][i] = fmaf(p, vx[i], o[r][i]);
            }
        }
        __syncwarp();
    }
#pragma unroll
    for (int r = 0; r < PA_ROWS; ++r) {
#pragma unroll
        for (int of = 16; of > 0; of >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], of);
        if (lane == 0) { s_m[warp][r] = m[r]; s_l[warp][r] = l[r]; }
#pragma unroll
        for (int i = 0; i < DL; ++i) s_o[warp][r][lane * DL + i] = o[r][i];
    }
    __syncthreads();
    for (int i = tid; i < PA_ROWS * D; i += 128) {
        const int r = i / D, d = i % D, row = row0 + r;
        if (row >= n_rows) break;
        float mx = s_m[0][r];
        for (int w = 1; w < 4; ++w) mx = fmaxf(mx, s_m[w][r]);
        const float base = mx == -INFINITY ? 0.0f : mx;
        float sum = 0.0f, acc = 0.0f;
        for (int w = 0; w < 4; ++w) { const float f = exp2f(s_m[w][r] - base); sum += f * s_l[w][r]; if (f != 0.0f) acc += f * s_o[w][r][d]; }
        const int t = row / a.group, h = kvh * a.group + row % a.group;
        const int64_t out = (s.tok0 + t) * a.n_head + h;
        if (a.n_split == 1) {
            ((Q *) (a.dst + (s.tok0 + t) * a.nb_dst_tok + h * a.nb_dst_head))[d] = (Q) (sum == 0.0f ? 0.0f : acc / sum);
            if (a.lse && d == 0) a.lse[out] = sum == 0.0f ? -INFINITY : mx * 0.69314718f + logf(sum);
        } else {
            float * p = a.part + (split * a.n_tok * a.n_head + out) * (D + 2);
            p[d] = acc;
            if (d == 0) { p[D] = mx; p[D + 1] = sum; }
        }
    }
}

// joins the splits of a row: one warp per row
template <typename Q, int D>
__global__ void __launch_bounds__(128)
k_paged_join(PaArgs a) {
    chain_release();
    chain_wait();
    constexpr int DL = D / 32;
    const int lane = threadIdx.x & 31;
    const int seq = blockIdx.y;
    const PaSeq s = pa_seq(a, seq);
    for (int64_t w = (int64_t) blockIdx.x * 4 + (threadIdx.x >> 5); w < (int64_t) s.n_new * a.n_head; w += (int64_t) gridDim.x * 4) {
        const int t = (int) (w / a.n_head), h = (int) (w - (int64_t) t * a.n_head);
        const int64_t out = (s.tok0 + t) * a.n_head + h;
        const int row = t * a.group + h % a.group, row0 = row / PA_ROWS * PA_ROWS;
        const int last_t = (min(row0 + PA_ROWS, s.n_new * a.group) - 1) / a.group;
        const int reach = a.causal ? min(s.len, max(s.len - s.n_new + last_t + 1, 0)) : s.len;
        const int n = max(1, (reach + a.chunk - 1) / a.chunk);
        const float * p = a.part + out * (D + 2);
        const int64_t step = a.n_tok * a.n_head * (D + 2);
        float mx = -INFINITY;
        for (int i = lane; i < n; i += 32) mx = fmaxf(mx, p[i * step + D]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float base = mx == -INFINITY ? 0.0f : mx;
        float sum = 0.0f, acc[DL] = {};
        for (int i = 0; i < n; ++i) {
            const float f = exp2f(p[i * step + D] - base);
            sum += f * p[i * step + D + 1];                 // NaN of a split without a finite maximum stays NaN
            if (f == 0.0f) continue;
#pragma unroll
            for (int j = 0; j < DL; ++j) acc[j] += f * p[i * step + lane * DL + j];
        }
#pragma unroll
        for (int j = 0; j < DL; ++j)
            ((Q *) (a.dst + (s.tok0 + t) * a.nb_dst_tok + h * a.nb_dst_head))[lane * DL + j] = (Q) (sum == 0.0f ? 0.0f : acc[j] / sum);
        if (a.lse && lane == 0) a.lse[out] = sum == 0.0f ? -INFINITY : mx * 0.69314718f + logf(sum);
    }
}

// ---- host ----------------------------------------------------------------------------------------
static bool pa_args_ok(const b200_page_pool * p, const b200_paged_attn_args * a, bool attn) {
    if (!a || !b200_pool_ok(p, true) || a->layer < 0 || a->layer >= p->n_layer) return false;
    if (a->n_seq < 0 || a->n_seq > 65535 || a->n_tok < 0 || a->n_tok > 0x7fffffff || a->max_new < 0 || a->max_len < 0 || a->max_len >= (1ll << 30)) return false;
    if (a->q_type != B200_TYPE_F32 && a->q_type != p->type) return false;
    if (a->n_seq == 0 || a->n_tok == 0 || a->max_new == 0) return true;
    if (!a->tables || a->table_stride < 1 || !a->lens || !a->q_start) return false;
    if (!a->k_new != !a->v_new || (!attn && !a->k_new)) return false;
    const int64_t size = a->q_type == B200_TYPE_F32 ? 4 : 2, row = size * p->head_dim;
    if (a->k_new && (((uintptr_t) a->k_new | (uintptr_t) a->v_new | (uintptr_t) a->nb_new_tok | (uintptr_t) a->nb_new_head) % 16 ||
                     a->nb_new_tok < 0 || a->nb_new_head < 0)) return false;
    if (!attn) return true;
    if (!a->q || !a->dst || a->n_head < 1 || a->n_head % p->n_head_kv || a->n_head > 4096) return false;
    if (((uintptr_t) a->q | (uintptr_t) a->dst | (uintptr_t) a->nb_q_tok | (uintptr_t) a->nb_q_head | (uintptr_t) a->nb_dst_tok | (uintptr_t) a->nb_dst_head) % 16) return false;
    if (a->nb_q_tok < 0 || a->nb_q_head < 0 || (a->n_head > 1 && a->nb_dst_head < row) || (a->n_tok > 1 && a->nb_dst_tok < row)) return false;
    return a->scale == a->scale && a->scale - a->scale == 0.0f;        // finite
}

// keys per split and number of splits: enough CTAs to fill the device, no split shorter than a few blocks of keys
static void pa_plan(const b200_page_pool * p, const b200_paged_attn_args * a, int * n_split, int * chunk) {
    const int64_t group = a->n_head / p->n_head_kv;
    const int64_t new_max = a->max_new < a->n_tok ? a->max_new : a->n_tok;
    const int64_t ctas = (new_max * group + PA_ROWS - 1) / PA_ROWS * p->n_head_kv * a->n_seq;
    int64_t want = (148 * 8 + ctas - 1) / ctas, most = (a->max_len + 127) / 128;
    if (want > most) want = most;
    if (want > 64) want = 64;
    if (want < 1) want = 1;
    int64_t c = ((a->max_len + want - 1) / want + 31) / 32 * 32;
    if (c < 32) c = 32;
    *chunk = (int) c;
    *n_split = (int) ((a->max_len + c - 1) / c);
    if (*n_split < 1) *n_split = 1;
}

extern "C" int64_t b200_paged_attn_workspace(const b200_page_pool * pool, const b200_paged_attn_args * a) {
    if (!a || !b200_pool_ok(pool, true) || a->n_tok < 1 || a->n_seq < 1 || a->max_new < 1 || a->max_len < 0 || a->max_len >= (1ll << 30) ||
        a->n_head < 1 || a->n_head % pool->n_head_kv) return 0;
    int n_split, chunk;
    pa_plan(pool, a, &n_split, &chunk);
    return n_split == 1 ? 0 : (int64_t) n_split * a->n_tok * a->n_head * (pool->head_dim + 2) * 4;
}

static PaArgs pa_pack(const b200_page_pool * p, const b200_paged_attn_args * a) {
    PaArgs k = {};
    k.q = (const char *) a->q; k.nb_q_tok = a->nb_q_tok; k.nb_q_head = a->nb_q_head;
    k.dst = (char *) a->dst; k.nb_dst_tok = a->nb_dst_tok; k.nb_dst_head = a->nb_dst_head;
    k.k = (const char *) p->k + a->layer * p->nb_layer; k.v = (const char *) p->v + a->layer * p->nb_layer;
    k.nb_page = p->nb_page; k.nb_tok = p->nb_tok; k.nb_head = p->nb_head;
    k.tables = a->tables; k.table_stride = a->table_stride; k.lens = a->lens; k.q_start = a->q_start;
    k.lse = a->lse; k.part = (float *) a->workspace; k.n_tok = a->n_tok; k.max_len = a->max_len;
    k.n_pages = p->n_pages; k.page_size = p->page_size; k.n_head = a->n_head; k.n_head_kv = p->n_head_kv;
    k.group = a->n_head / p->n_head_kv; k.causal = a->causal != 0;
    k.max_new = (int) (a->max_new < a->n_tok ? a->max_new : a->n_tok);
    k.scale_log2 = a->scale * 1.44269504f;
    return k;
}

extern "C" int b200_paged_store(const b200_page_pool * pool, const b200_paged_attn_args * a, void * stream) {
    if (!pa_args_ok(pool, a, false)) return B200_ERR_ARG;
    if (a->n_seq == 0 || a->n_tok == 0 || a->max_new == 0) return 0;
    b200_paged_attn_args b = *a;
    if (b.n_head < 1) b.n_head = pool->n_head_kv;
    const PaArgs k = pa_pack(pool, &b);
    const PaNew x = { (const char *) a->k_new, (const char *) a->v_new, a->nb_new_tok, a->nb_new_head };
    const int vec_head = pool->head_dim / 8;
    int64_t n = ((int64_t) k.max_new * 2 * pool->n_head_kv * vec_head + 255) / 256;
    const int64_t most = (148 * 8 + a->n_seq - 1) / a->n_seq;
    if (n > most) n = most;
    const bool f32 = a->q_type == B200_TYPE_F32, h = pool->type == B200_TYPE_F16;
    auto f = h ? (f32 ? k_paged_store<__half, true> : k_paged_store<__half, false>) : (f32 ? k_paged_store<__nv_bfloat16, true> : k_paged_store<__nv_bfloat16, false>);
    const cudaError_t e = launch_chained(f, dim3((unsigned) n, (unsigned) a->n_seq), dim3(256), 0, as_stream(stream), k, x, vec_head);
    if (e != cudaSuccess) return (int) e;
    B200_RETURN_LAST();
}

template <typename Q, typename KV, int D>
static cudaError_t pa_launch(PaArgs & k, int n_seq, cudaStream_t st) {
    const int64_t tiles = ((int64_t) k.max_new * k.group + PA_ROWS - 1) / PA_ROWS;
    cudaError_t e = launch_chained(k_paged_attn<Q, KV, D>, dim3((unsigned) tiles, (unsigned) k.n_head_kv, (unsigned) (n_seq * k.n_split)), dim3(128), 0, st, k);
    if (e != cudaSuccess) return e;
    B200_LAUNCHED();
    if (k.n_split == 1) return cudaGetLastError();
    int64_t n = ((int64_t) k.max_new * k.n_head + 3) / 4;
    if (n > 4096) n = 4096;
    e = launch_chained(k_paged_join<Q, D>, dim3((unsigned) n, (unsigned) n_seq), dim3(128), 0, st, k);
    if (e == cudaSuccess) B200_LAUNCHED();
    return e;
}

extern "C" int b200_paged_attn(const b200_page_pool * pool, const b200_paged_attn_args * a, void * stream) {
    if (!pa_args_ok(pool, a, true)) return B200_ERR_ARG;
    if (a->n_seq == 0 || a->n_tok == 0 || a->max_new == 0) return 0;
    PaArgs k = pa_pack(pool, a);
    pa_plan(pool, a, &k.n_split, &k.chunk);
    const int64_t need = b200_paged_attn_workspace(pool, a);
    if (need && (!a->workspace || (uintptr_t) a->workspace % 16 || a->workspace_bytes < need)) return B200_ERR_ARG;
    if ((int64_t) a->n_seq * k.n_split > 65535) return B200_ERR_ARG;
    if (a->k_new) {
        const int rc = b200_paged_store(pool, a, stream);
        if (rc) return rc;
    }
    const cudaStream_t st = as_stream(stream);
    const bool f32 = a->q_type == B200_TYPE_F32, h = pool->type == B200_TYPE_F16;
    cudaError_t e;
    if (pool->head_dim == 64)
        e = f32 ? (h ? pa_launch<float, __half, 64>(k, a->n_seq, st) : pa_launch<float, __nv_bfloat16, 64>(k, a->n_seq, st))
                : (h ? pa_launch<__half, __half, 64>(k, a->n_seq, st) : pa_launch<__nv_bfloat16, __nv_bfloat16, 64>(k, a->n_seq, st));
    else
        e = f32 ? (h ? pa_launch<float, __half, 128>(k, a->n_seq, st) : pa_launch<float, __nv_bfloat16, 128>(k, a->n_seq, st))
                : (h ? pa_launch<__half, __half, 128>(k, a->n_seq, st) : pa_launch<__nv_bfloat16, __nv_bfloat16, 128>(k, a->n_seq, st));
    return (int) e;
}
