// Attention of a chunk of new tokens over a paged key/value cache, single tokens included, and the store that precedes it.
// The reference has one dense cache per state (whisper_kv_cache, src/whisper.cpp:1000-1200) and decodes through
// ggml_compute_forward_flash_attn_ext_f16 (ggml/src/ggml-cpu/ops.cpp:6638-6851); this operator is defined by its formula
// (include/b200_whisper.h), with 32-bit scores, weights' sums and accumulators.
#include "paged_attn.cuh"

bool b200_pool_ok(const b200_page_pool * p, bool data);    // k_pages.cu

struct PaNew { const char * k; const char * v; int64_t nb_tok, nb_head; };      // new rows to be stored (type of q)

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


// a warp per token, 16 bytes of the pool a lane; f32 is rounded to the pool's type (to nearest even: the cache's precision), 16-bit values are
// copied.  Bound by memory: every value is read and written once
template <typename KV, bool F32>
__global__ void __launch_bounds__(256)
k_paged_store(const __grid_constant__ PaArgs a, const __grid_constant__ PaNew x, int log_vec) {
    chain_wait();                                         // in this order: once all CTAs have released, all that came before this launch is there,
    chain_release();                                      // and the attention behind it may read its queries and tables at once (32 ragged prompts: 36.1 -> 34.2 us)
    const int failed = pa_failed(a);
    const PaSeq s = pa_seq(a, blockIdx.y);
    if (failed) return;
    const int lane = threadIdx.x & 31, per_tok = 2 * a.n_head_kv << log_vec, mask = (1 << log_vec) - 1;
    for (int t = blockIdx.x * 8 + (threadIdx.x >> 5); t < s.n_new; t += gridDim.x * 8) {
        const int pos = s.len - s.n_new + t;
        if (pos < 0) continue;
        const int page = a.tables[blockIdx.y * a.table_stride + pos / a.page_size];
        if (page < 0 || page >= a.n_pages) continue;
        const int64_t at = page * a.nb_page + (pos % a.page_size) * a.nb_tok, from = (s.tok0 + t) * x.nb_tok;
#pragma unroll 4
        for (int r = lane; r < per_tok; r += 32) {
            const int c = r & mask, hv = r >> log_vec;
            const bool v = hv >= a.n_head_kv;
            const int h = v ? hv - a.n_head_kv : hv;
            const char * src = (v ? x.v : x.k) + from + h * x.nb_head;
            uint4 q;
            if (F32) {
                float f[8];
                *(float4 *) f = ((const float4 *) src)[2 * c];
                *(float4 *) (f + 4) = ((const float4 *) src)[2 * c + 1];
                q = pa_pack8<KV>(f);
            } else q = ((const uint4 *) src)[c];
            *(uint4 *) ((char *) (v ? a.v : a.k) + at + h * a.nb_head + c * 16) = q;
        }
    }
}

// ---- attention of few rows, and of f32 queries ---------------------------------------------------
// A row is one query token of one query head; the rows of a key/value head are numbered token * group + head in group.  A CTA
// takes 16 rows of one sequence and key/value head over one split of the keys - the 16 rows of an mma.sync m16n8k16 - and each of
// its four warps streams every fourth block of keys (4 KB of K, 4 KB of V) through its own shared-memory ring (two blocks deep, K and
// V separate cp.async groups), so nothing in the loop waits for another warp.  Running maximum and sum per row; the warps are joined through
// shared memory at the end, the splits by k_paged_join.  Bound by the stream of K and V.  Rings of 16 KB
// put three CTAs on an SM; with twice the block, and one CTA, 64 sequences of up to 8192 keys (head_dim 128) took 292 us instead of 189.
//
// F32 queries: q and the weights are written as sums of two f16 (the second scaled by 2^11, q scaled by a power of two per row
// so that no part underflows) or three bf16 values, which hold 22 or 24 bits of them, and each part is multiplied on the tensor
// pipe; products of a block are added to the f32 accumulator by FADD, because the tensor pipe's own accumulation truncates.
#define PA_ROWS  16
#define PA_BLOCK 4096                            // bytes of a block of K or V: 32 keys of 64 or 16 of 128 dimensions
#define PA_WARPS 4
#define PA_WIDE_MIN_ROWS 64                      // f32 queries: with more rows a head, and this many tiles of 16 rows, k_paged_attn_wide
#define PA_WIDE_MIN_ITEMS (6 * 148)

template <typename T> struct PaPack;
template <> struct PaPack<__half> {
    static __device__ __forceinline__ uint32_t two(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *(const uint32_t *) &h; }
    static __device__ __forceinline__ float2 back(uint32_t w) { return __half22float2(*(const __half2 *) &w); }
    static __device__ __forceinline__ uint32_t odd(uint32_t w) { return ((w & 0x7c00u) == 0x7c00u ? 0xffffu : 0u) | ((w & 0x7c000000u) == 0x7c000000u ? 0xffff0000u : 0u); }
    static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t * a, uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
template <> struct PaPack<__nv_bfloat16> {
    static __device__ __forceinline__ uint32_t two(float a, float b) { const __nv_bfloat162 h = __floats2bfloat162_rn(a, b); return *(const uint32_t *) &h; }
    static __device__ __forceinline__ float2 back(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
    static __device__ __forceinline__ uint32_t odd(uint32_t w) { return ((w & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((w & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u); }
    static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t * a, uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};

// parts of an f32 operand; `lift` is the factor between one part and the next (1: none)
template <typename Q, typename KV> struct PaParts { static constexpr int n = 1; static constexpr float lift = 1.0f; };
template <> struct PaParts<float, __half>        { static constexpr int n = 2; static constexpr float lift = 2048.0f; };
template <> struct PaParts<float, __nv_bfloat16> { static constexpr int n = 3; static constexpr float lift = 1.0f; };

template <typename Q, typename KV>
__device__ __forceinline__ void pa_parts(float a, float b, uint32_t (&out)[PaParts<Q, KV>::n]) {
    using P = PaParts<Q, KV>;
#pragma unroll
    for (int i = 0; i < P::n; ++i) {
        out[i] = PaPack<KV>::two(a, b);
        const float2 f = PaPack<KV>::back(out[i]);
        a = (a - f.x) * P::lift; b = (b - f.y) * P::lift;
    }
}

__device__ __forceinline__ uint32_t pa_smem(const void * p) { return (uint32_t) __cvta_generic_to_shared(p); }
__device__ __forceinline__ void pa_cp16(uint32_t dst, const void * src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void pa_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void pa_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory"); }
__device__ __forceinline__ void pa_ldm(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3},[%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void pa_ldm_t(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3},[%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}

// 16 rows of a warp and one block of keys after another.  Of the rows a lane has two: lane / 4 and lane / 4 + 8
template <typename Q, typename KV, int D> struct PaTile {
    using P = PaPack<KV>;
    static constexpr int NP = PaParts<Q, KV>::n, NC = D / 8, KS = D / 16, KEYS = PA_BLOCK / (2 * D), NK = KEYS / 8;      // parts, 16-byte chunks and MMA steps of a head; keys of a block, MMA columns of its scores
    static constexpr float LIFT = PaParts<Q, KV>::lift;
    // f16 has all its bits from 2^-14 on and nothing below 2^-25: the weights, 1 at the running maximum, enter the product with V times 2^14, so that
    // many small ones beside a large one count (131072 keys of weight 2^-26 and one of 1 and value 0: the result was 0 instead of 0.002)
    static constexpr float RAISE = std::is_same<KV, __half>::value ? 16384.0f : 1.0f;
    uint32_t qf[NP][KS][4], pf[NP][NK / 2][4];
    float fa, fb, o[NC][4], sc[NK][4], ma, mb, la, lb;
    int last_a, last_b, first_last;                       // keys up to last_*: seen by the row; up to first_last: by every row

    __device__ __forceinline__ void start(const PaArgs & a, const PaSeq & s, int kvh, int row0, int n_rows) {
        const int lane = threadIdx.x & 31;
        const int ra = row0 + (lane >> 2), rb = ra + 8;
        last_a = ra >= n_rows ? -1 : a.causal ? s.len - s.n_new + ra / a.group : s.len - 1;
        last_b = rb >= n_rows ? -1 : a.causal ? s.len - s.n_new + rb / a.group : s.len - 1;
        first_last = a.causal ? s.len - s.n_new + row0 / a.group : s.len - 1;
        fa = fb = a.scale_log2;
        ma = mb = -INFINITY; la = lb = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c) o[c][0] = o[c][1] = o[c][2] = o[c][3] = 0.0f;
        {
            const int ia = min(ra, n_rows - 1), ib = min(rb, n_rows - 1);
            const Q * qa = (const Q *) (a.q + (s.tok0 + ia / a.group) * a.nb_q_tok + (kvh * a.group + ia % a.group) * a.nb_q_head) + (lane & 3) * 2;
            const Q * qb = (const Q *) (a.q + (s.tok0 + ib / a.group) * a.nb_q_tok + (kvh * a.group + ib % a.group) * a.nb_q_head) + (lane & 3) * 2;
            if constexpr (NP == 1) {
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    qf[0][i][0] = *(const uint32_t *) (qa + 16 * i);     qf[0][i][1] = *(const uint32_t *) (qb + 16 * i);
                    qf[0][i][2] = *(const uint32_t *) (qa + 16 * i + 8); qf[0][i][3] = *(const uint32_t *) (qb + 16 * i + 8);
                }
            } else {
                float2 x[KS][4];
                float xa = 0.0f, xb = 0.0f;
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    x[i][0] = *(const float2 *) (qa + 16 * i);     x[i][1] = *(const float2 *) (qb + 16 * i);
                    x[i][2] = *(const float2 *) (qa + 16 * i + 8); x[i][3] = *(const float2 *) (qb + 16 * i + 8);
                    xa = fmaxf(fmaxf(xa, fmaxf(fabsf(x[i][0].x), fabsf(x[i][0].y))), fmaxf(fabsf(x[i][2].x), fabsf(x[i][2].y)));
                    xb = fmaxf(fmaxf(xb, fmaxf(fabsf(x[i][1].x), fabsf(x[i][1].y))), fmaxf(fabsf(x[i][3].x), fabsf(x[i][3].y)));
                }
                float sa = 1.0f, sb = 1.0f;
                if constexpr (LIFT != 1.0f) {                // powers of two that bring the row's largest value to [1, 2)
#pragma unroll
                    for (int o = 1; o < 4; o <<= 1) { xa = fmaxf(xa, __shfl_xor_sync(0xffffffffu, xa, o)); xb = fmaxf(xb, __shfl_xor_sync(0xffffffffu, xb, o)); }
                    auto inverse = [](float m) { const int e = (int) (__float_as_uint(m) >> 23); return e == 0 || e == 255 ? 1.0f : __uint_as_float((uint32_t) max(1, 254 - e) << 23); };
                    sa = inverse(xa); sb = inverse(xb);
                    fa = a.scale_log2 / sa; fb = a.scale_log2 / sb;
                }
#pragma unroll
                for (int i = 0; i < KS; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float f = j & 1 ? sb : sa;
                        uint32_t w[NP];
                        pa_parts<Q, KV>(x[i][j].x * f, x[i][j].y * f, w);
#pragma unroll
                        for (int n = 0; n < NP; ++n) qf[n][i][j] = w[n];
                    }
            }
        }
    }
    // of the block at kb
    __device__ __forceinline__ void scores(uint32_t kb) {
        const int lane = threadIdx.x & 31;
        float part[NP][NK][4] = {};
#pragma unroll
        for (int h = 0; h < KS / 2; ++h) {
            uint32_t b[NK][4];
#pragma unroll
            for (int j = 0; j < NK; ++j) pa_ldm(b[j], kb + (8 * j + (lane & 7)) * D * 2 + (((4 * h + (lane >> 3)) ^ (lane & 7)) << 4));
#pragma unroll
            for (int n = 0; n < NP; ++n)
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int j = 0; j < NK; ++j) P::mma(part[n][j], qf[n][2 * h + u], b[j][2 * u], b[j][2 * u + 1]);
        }
#pragma unroll
        for (int j = 0; j < NK; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float v = part[NP - 1][j][e];
#pragma unroll
                for (int n = NP - 2; n >= 0; --n) v = part[n][j][e] + v * (1.0f / LIFT);
                sc[j][e] = v;
            }
    }
    // masks (edge: some row does not see the whole block), running maximum and sum, weights in parts, o to the new maximum
    __device__ __forceinline__ void weights(int key0, int k1, bool edge) {
        const int lane = threadIdx.x & 31;
        float xa = -INFINITY, xb = -INFINITY;
#pragma unroll
        for (int j = 0; j < NK; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                sc[j][e] *= fa; sc[j][e + 2] *= fb;
                if (edge) {
                    const int key = key0 + 8 * j + (lane & 3) * 2 + e;
                    if (key >= k1 || key > last_a) sc[j][e] = -INFINITY;
                    if (key >= k1 || key > last_b) sc[j][e + 2] = -INFINITY;
                }
                xa = fmaxf(xa, sc[j][e]); xb = fmaxf(xb, sc[j][e + 2]);
            }
#pragma unroll
        for (int of = 1; of < 4; of <<= 1) { xa = fmaxf(xa, __shfl_xor_sync(0xffffffffu, xa, of)); xb = fmaxf(xb, __shfl_xor_sync(0xffffffffu, xb, of)); }
        xa = fmaxf(xa, ma); xb = fmaxf(xb, mb);
        const float ba = xa == -INFINITY ? 0.0f : xa, bb = xb == -INFINITY ? 0.0f : xb;
        const float ca = pa_exp2(ma - ba), cb = pa_exp2(mb - bb);
        ma = xa; mb = xb;
        la *= ca; lb *= cb;
#pragma unroll
        for (int j = 0; j < NK; ++j) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                sc[j][e] = pa_exp2(sc[j][e] - ba); sc[j][e + 2] = pa_exp2(sc[j][e + 2] - bb);
                la += sc[j][e]; lb += sc[j][e + 2];
            }
            uint32_t w[NP];
            pa_parts<Q, KV>(sc[j][0] * RAISE, sc[j][1] * RAISE, w);
#pragma unroll
            for (int n = 0; n < NP; ++n) pf[n][j >> 1][(j & 1) * 2] = w[n];
            pa_parts<Q, KV>(sc[j][2] * RAISE, sc[j][3] * RAISE, w);
#pragma unroll
            for (int n = 0; n < NP; ++n) pf[n][j >> 1][(j & 1) * 2 + 1] = w[n];
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) { o[c][0] *= ca; o[c][1] *= ca; o[c][2] *= cb; o[c][3] *= cb; }
    }
    // o += weights * the block at vb
    __device__ __forceinline__ void values(const char * smem, uint32_t vb, int key0, int k1, bool edge) {
        const int lane = threadIdx.x & 31;
        uint32_t odd = 0;
#pragma unroll
        for (int c = 0; c < NC / 2; ++c) {
            float part[NP][2][4] = {};
#pragma unroll
            for (int h = 0; h < NK / 2; ++h) {
                uint32_t b[4];
                pa_ldm_t(b, vb + (16 * h + (lane & 15)) * D * 2 + (((2 * c + (lane >> 4)) ^ (lane & 7)) << 4));
                if (edge) {                               // 0 * v is not 0 where v is infinite or NaN: such values are taken out here
#pragma unroll
                    for (int w = 0; w < 4; ++w) { const uint32_t x = P::odd(b[w]); odd |= x; b[w] &= ~x; }
                }
#pragma unroll
                for (int n = 0; n < NP; ++n) {
                    if constexpr (NP == 1) { P::mma(o[2 * c], pf[0][h], b[0], b[1]); P::mma(o[2 * c + 1], pf[0][h], b[2], b[3]); }
                    else { P::mma(part[n][0], pf[n][h], b[0], b[1]); P::mma(part[n][1], pf[n][h], b[2], b[3]); }
                }
            }
            if constexpr (NP > 1) {
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float v = part[NP - 1][u][e];
#pragma unroll
                        for (int n = NP - 2; n >= 0; --n) v = part[n][u][e] + v * (1.0f / LIFT);
                        o[2 * c + u][e] += v;
                    }
            }
        }
        if (edge && __any_sync(0xffffffffu, odd)) {       // ... and given back to the rows that see them
            for (int j = 0; j < min(KEYS, k1 - key0); ++j)
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const KV * v = (const KV *) (smem + (vb - pa_smem(smem)) + j * D * 2 + ((c ^ (j & 7)) << 4)) + (lane & 3) * 2;
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float x = (float) v[e];
                        if (!(fabsf(x) < INFINITY)) {
                            if (key0 + j <= last_a) o[c][e] += x;
                            if (key0 + j <= last_b) o[c][e + 2] += x;
                        }
                    }
                }
        }
    }
    __device__ __forceinline__ void finish() {
#pragma unroll
        for (int of = 1; of < 4; of <<= 1) { la += __shfl_xor_sync(0xffffffffu, la, of); lb += __shfl_xor_sync(0xffffffffu, lb, of); }
        if constexpr (RAISE != 1.0f) {
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[c][e] *= 1.0f / RAISE;
        }
    }
};

// How the work is dealt out.  Items are (sequence, key/value head, tile of 16 rows), numbered in that order; an item of a sequence of n keys
// is ceil(n / round) rounds of PA_WARPS blocks, at least one.  Either a CTA takes one item (a.stream = 0), or the rounds of all items are one
// line that is cut into a.stream equal parts, one per CTA: whatever the lengths, all CTAs end together.  On the line an item begins with
// PA_START rounds of nothing, the time that it takes to get its first keys.  A CTA then has up to two partial items, at the ends of its
// part; it leaves them in slots 0 (an item begun by another CTA) and 1, and k_paged_join puts them together.
// (64 sequences of 1 to 8192 keys: 224 us without it, 183 with 2, 181 with 4 or 8.)
#define PA_START 3
struct PaLine { int64_t total, before; };                 // rounds of all sequences, and of those before a given one
__device__ __forceinline__ int64_t pa_rounds(const PaArgs & a, const PaSeq & s, int round) {
    return (int64_t) ((s.n_new * a.group + PA_ROWS - 1) / PA_ROWS) * a.n_head_kv * (max(1, (s.len + round - 1) / round) + PA_START);
}
// this warp's lanes go over the sequences, a run of them each
__device__ __forceinline__ PaLine pa_line(const PaArgs & a, int round, int64_t target, int upto, int * seq_at, int64_t * rest) {
    const int lane = threadIdx.x & 31, per = (a.n_seq + 31) / 32, s0 = min(a.n_seq, lane * per), s1 = min(a.n_seq, s0 + per);
    int64_t mine = 0;
    for (int s = s0; s < s1; ++s) mine += pa_rounds(a, pa_seq(a, s), round);
    int64_t inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int64_t u = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += u; }
    PaLine l;
    l.total = __shfl_sync(0xffffffffu, inc, 31);
    l.before = 0;
    if (upto >= 0) {                                       // rounds before sequence `upto`
        int64_t b = inc - mine;
        if (upto >= s0 && upto < s1) for (int s = s0; s < upto; ++s) b += pa_rounds(a, pa_seq(a, s), round);
        l.before = __shfl_sync(0xffffffffu, b, upto / per);
    }
    if (seq_at) {                                          // the sequence that holds round target * total / a.stream
        const int64_t w = target * l.total / a.stream;
        const bool here = w >= inc - mine && w < inc;
        int s = s0;
        int64_t left = w - (inc - mine);
        if (here) for (; s < s1; ++s) { const int64_t r = pa_rounds(a, pa_seq(a, s), round); if (left < r) break; left -= r; }
        const unsigned who = __ballot_sync(0xffffffffu, here);
        const int src = who ? __ffs(who) - 1 : 0;
        *seq_at = who ? __shfl_sync(0xffffffffu, s, src) : a.n_seq;
        *rest = __shfl_sync(0xffffffffu, left, src);
    }
    return l;
}


template <typename Q, typename KV, int D, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, WARPS > PA_WARPS ? 1 : PaParts<Q, KV>::n == 1 ? 3 : 2)
k_paged_attn(const __grid_constant__ PaArgs a, const __grid_constant__ PaNew nw) {
    using P = PaPack<KV>;
    constexpr int NP = PaParts<Q, KV>::n, NC = D / 8, BLOCK = PA_BLOCK, KEYS = PaTile<Q, KV, D>::KEYS, ROUND = KEYS * WARPS;
    extern __shared__ __align__(16) char smem[];
    // The successor is let in only when CTAs end: brought in early, the CTAs of the join and of the next call took the places of this kernel's
    // own (111 sequences of 4096 keys: 121 us a call, 85 without).
    chain_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);      // the shuffle tells the compiler that the warp agrees
    int seq, kvh, tile, at = 0;                           // the item, and where in it (on the line) this CTA begins
    int64_t todo = 1ll << 60;                             // what is left of this CTA's part
    const int failed = pa_failed(a);
    if (a.stream) {
        int64_t rest;
        const PaLine l = pa_line(a, ROUND, blockIdx.x, -1, &seq, &rest);
        todo = ((int64_t) blockIdx.x + 1) * l.total / a.stream - (int64_t) blockIdx.x * l.total / a.stream;
        if (seq >= a.n_seq || todo == 0 || failed) return;
        const PaSeq s = pa_seq(a, seq);
        const int rounds = max(1, (s.len + ROUND - 1) / ROUND), tiles = (s.n_new * a.group + PA_ROWS - 1) / PA_ROWS;
        const int64_t item = rest / (rounds + PA_START);
        at = (int) (rest - item * (rounds + PA_START));
        kvh = (int) (item / tiles);
        tile = (int) (item - (int64_t) kvh * tiles);
    } else { seq = blockIdx.z; kvh = blockIdx.y; tile = gridDim.x - 1 - blockIdx.x; }      // the longest tiles first
    for (;;) {
    const PaSeq s = pa_seq(a, seq);
    const int n_rows = s.n_new * a.group, row0 = tile * PA_ROWS;
    if (!a.stream && (row0 >= n_rows || failed)) return;
    const int rounds = max(1, (s.len + ROUND - 1) / ROUND), steps = (int) min((int64_t) (rounds + PA_START - at), todo);
    const int first_round = max(0, at - PA_START), n_round = max(0, at + steps - PA_START) - first_round;
    const int k0 = first_round * ROUND, k1 = min(pa_reach(a, s, row0), k0 + n_round * ROUND);
    const bool whole = n_round == rounds;
    if (n_round > 0) {

    const char * kp = a.k + kvh * a.nb_head, * vp = a.v + kvh * a.nb_head;
    const int32_t * table = a.tables + seq * a.table_stride;
    const uint32_t ring = pa_smem(smem) + warp * 4 * BLOCK;             // K0 K1 V0 V1
    const int n_block = k1 > k0 ? (k1 - k0 + KEYS - 1) / KEYS : 0, n_mine = (n_block - warp + WARPS - 1) / WARPS;
    auto key_of = [&](int i) { return k0 + (i * WARPS + warp) * KEYS + lane; };
    auto page_of = [&](int i) { const int key = key_of(i); return i < n_mine && lane < KEYS && key < k1 ? table[key / a.page_size] : -1; };
    const int new0 = nw.k ? s.len - s.n_new : 1 << 30;    // from here on K and V come from the new rows
    auto at_of = [&](int i, int page) -> int64_t {       // this lane's key's place in the pool, -1: none
        int64_t at = page >= 0 && page < a.n_pages ? page * a.nb_page + (key_of(i) % a.page_size) * a.nb_tok : -1;
        asm volatile("" : "+l"(at));                     // kept: the compiler computes it again for every chunk otherwise, division included
        return at;
    };
    // a block of K or V into its stage.  New rows are read where the caller has them; the last tile, which
    // sees them all, also writes them to their pages
    auto load = [&](int i, int64_t at, bool is_v, uint32_t dst) {
        if (i < n_mine) {
            const char * base = is_v ? vp : kp;
            const int key0 = k0 + (i * WARPS + warp) * KEYS;
            if (key0 + KEYS <= new0) {
#pragma unroll
                for (int c = 0; c < NC * KEYS / 32; ++c) {
                    const int x = c * 32 + lane, r = x / NC, ch = x % NC;
                    const int64_t off = __shfl_sync(0xffffffffu, at, r);
                    pa_cp16(dst + r * D * 2 + ((ch ^ (r & 7)) << 4), base + (off < 0 ? 0 : off + ch * 16), off >= 0);
                }
            } else {
#pragma unroll 2
                for (int c = 0; c < NC * KEYS / 32; ++c) {
                    const int x = c * 32 + lane, r = x / NC, ch = x % NC;
                    const int64_t off = __shfl_sync(0xffffffffu, at, r);
                    const uint32_t d = dst + r * D * 2 + ((ch ^ (r & 7)) << 4);
                    if (key0 + r < new0 || off < 0) { pa_cp16(d, base + (off < 0 ? 0 : off + ch * 16), off >= 0); continue; }
                    const char * src = (is_v ? nw.v : nw.k) + (s.tok0 + key0 + r - new0) * nw.nb_tok + kvh * nw.nb_head;
                    uint4 q;
                    if constexpr (NP > 1) {
                        float f[8];
                        *(float4 *) f = ((const float4 *) src)[2 * ch];
                        *(float4 *) (f + 4) = ((const float4 *) src)[2 * ch + 1];
                        q = pa_pack8<KV>(f);
                    } else q = ((const uint4 *) src)[ch];
                    *(uint4 *) (smem + (d - pa_smem(smem))) = q;
                    if ((tile + 1) * PA_ROWS >= n_rows) *(uint4 *) (const_cast<char *>(base) + off + ch * 16) = q;
                }
            }
        }
        pa_commit();
    };
    int64_t at_next;
    {
        const int p0 = page_of(0), p1 = page_of(1);
        const int64_t at0 = at_of(0, p0), at1 = at_of(1, p1);
        load(0, at0, false, ring); load(0, at0, true, ring + 2 * BLOCK);
        load(1, at1, false, ring + BLOCK); load(1, at1, true, ring + 3 * BLOCK);
    }
    int page_next = page_of(2);

    PaTile<Q, KV, D> t;
    t.start(a, s, kvh, row0, n_rows);
    for (int i = 0; i < n_mine; ++i) {
        const uint32_t kb = ring + (i & 1) * BLOCK, vb = kb + 2 * BLOCK;
        const int key0 = k0 + (i * WARPS + warp) * KEYS;
        at_next = at_of(i + 2, page_next);
        page_next = page_of(i + 3);
        pa_wait<3>();
        __syncwarp();
        t.scores(kb);
        __syncwarp();
        load(i + 2, at_next, false, kb);
        const bool edge = key0 + KEYS - 1 > t.first_last || key0 + KEYS > k1;
        t.weights(key0, k1, edge);
        pa_wait<3>();
        __syncwarp();
        t.values(smem, vb, key0, k1, edge);
        __syncwarp();
        load(i + 2, at_next, true, vb);
    }
    pa_wait<0>();
    t.finish();
    __syncthreads();
    // join of the four warps: [warp][row] maxima and sums, [warp][row][D + 4] accumulators over the rings
    float * sm = (float *) smem, * sl = sm + WARPS * PA_ROWS, * so = sl + WARPS * PA_ROWS;
    constexpr int LD = D + 4;
    {
        const int wa = warp * PA_ROWS + (lane >> 2), wb = wa + 8;
        if ((lane & 3) == 0) { sm[wa] = t.ma; sm[wb] = t.mb; sl[wa] = t.la; sl[wb] = t.lb; }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            *(float2 *) (so + wa * LD + c * 8 + (lane & 3) * 2) = make_float2(t.o[c][0], t.o[c][1]);
            *(float2 *) (so + wb * LD + c * 8 + (lane & 3) * 2) = make_float2(t.o[c][2], t.o[c][3]);
        }
    }
    __syncthreads();
    const int rows = min(PA_ROWS, n_rows - row0);
    for (int i = tid; i < rows * (D / 4); i += 32 * WARPS) {
        const int r = i / (D / 4), d = i % (D / 4) * 4, row = row0 + r;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) mx = fmaxf(mx, sm[w * PA_ROWS + r]);
        const float base = mx == -INFINITY ? 0.0f : mx;
        float sum = 0.0f, x[4] = {};
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float f = pa_exp2(sm[w * PA_ROWS + r] - base);
            sum += f * sl[w * PA_ROWS + r];              // NaN of a warp without a finite maximum stays NaN
            const float4 v = *(const float4 *) (so + (w * PA_ROWS + r) * LD + d);      // 0 * infinite is NaN, as it has to be
            x[0] += f * v.x; x[1] += f * v.y; x[2] += f * v.z; x[3] += f * v.w;
        }
        const int tok = row / a.group, h = kvh * a.group + row % a.group;
        const int64_t out = (s.tok0 + tok) * a.n_head + h;
        if (whole) {
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            char * dst = a.dst + (s.tok0 + tok) * a.nb_dst_tok + h * a.nb_dst_head + d * sizeof(Q);
            if constexpr (NP == 1) *(uint2 *) dst = make_uint2(P::two(x[0] * inv, x[1] * inv), P::two(x[2] * inv, x[3] * inv));
            else *(float4 *) dst = make_float4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
            if (a.lse && d == 0) a.lse[out] = sum == 0.0f ? -INFINITY : mx * 0.69314718f + logf(sum);
        } else {
            float * p = a.part + (((int64_t) blockIdx.x * 2 + (first_round == 0)) * PA_ROWS + r) * (D + 4);
            *(float4 *) (p + d) = make_float4(x[0], x[1], x[2], x[3]);
            if (d == 0) { p[D] = mx; p[D + 1] = sum; }
        }
    }
    }
    // the next item of this CTA's part
    todo -= steps;
    if (!a.stream || todo == 0) return;
    at = 0;
    if (++tile * PA_ROWS >= n_rows) {
        tile = 0;
        if (++kvh == a.n_head_kv) {
            kvh = 0;
            do { if (++seq >= a.n_seq) return; } while (pa_seq(a, seq).n_new == 0);
        }
    }
    __syncthreads();                                      // the accumulators are read before the ring is filled again
    }
}

// F32 queries, many rows: the eight warps of a CTA have 16 rows each and share every block of keys (three stages of two blocks, one barrier
// a stage), so that K and V come from L2 once per 128 rows.  The rows of a warp are finished in its registers: no join.  Bound by
// issue: the parts' products, and the additions that keep them in f32.  Against 16 rows a CTA, head_dim 64, f16: 32 ragged prompts of up to 224
// tokens of 20 heads 103 -> 67 us; 4 chunks of 300 over 1000 keys, 12 heads (912 tiles of 16 rows) 63 -> 52; head_dim 128, chunks of 1024 over
// 4k keys 1391 -> 1210.  With fewer tiles CTAs of 128 rows leave SMs idle: 16 chunks of 24 tokens x 4 heads x 8 (768 tiles) 95 -> 98, one
// prompt of 224 tokens of 20 heads 12.7 -> 18.0.
#define PA_WIDE 8
template <typename KV, int D>
__global__ void __launch_bounds__(32 * PA_WIDE, 1)
k_paged_attn_wide(const __grid_constant__ PaArgs a) {
    constexpr int NC = D / 8, KEYS = PaTile<float, KV, D>::KEYS, STAGE = 2 * KEYS, N = STAGE * NC / (32 * PA_WIDE), BYTES = 4 * PA_BLOCK, ROWS = PA_ROWS * PA_WIDE;
    extern __shared__ __align__(16) char smem[];
    chain_wait();                                         // no early release, as above
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const int seq = blockIdx.z, kvh = blockIdx.y, tile = gridDim.x - 1 - blockIdx.x;      // the longest tiles first
    const int failed = pa_failed(a);
    const PaSeq s = pa_seq(a, seq);
    const int n_rows = s.n_new * a.group, row0 = tile * ROWS, mine = row0 + warp * PA_ROWS;
    if (row0 >= n_rows || failed) return;
    auto reach = [&](int r1) { return a.causal ? min(s.len, max(s.len - s.n_new + (min(r1, n_rows) - 1) / a.group + 1, 0)) : s.len; };
    const int k1 = reach(row0 + ROWS), my_k1 = mine < n_rows ? reach(mine + PA_ROWS) : 0, n_stage = (k1 + STAGE - 1) / STAGE;
    const char * kp = a.k + kvh * a.nb_head, * vp = a.v + kvh * a.nb_head;
    const int32_t * table = a.tables + seq * a.table_stride;
    const uint32_t ring = pa_smem(smem);
    int page[N];
    auto look = [&](int i) {
#pragma unroll
        for (int c = 0; c < N; ++c) { const int key = i * STAGE + (c * 32 * PA_WIDE + tid) / NC; page[c] = i < n_stage && key < k1 ? table[key / a.page_size] : -1; }
    };
    auto load = [&](int i) {
        if (i < n_stage) {
            const uint32_t to = ring + i % 3 * BYTES;
#pragma unroll
            for (int c = 0; c < N; ++c) {
                const int x = c * 32 * PA_WIDE + tid, r = x / NC, ch = x % NC;
                const bool on = page[c] >= 0 && page[c] < a.n_pages;
                const int64_t off = on ? page[c] * a.nb_page + ((i * STAGE + r) % a.page_size) * a.nb_tok + ch * 16 : 0;
                const uint32_t d = to + r * D * 2 + ((ch ^ (r & 7)) << 4);
                pa_cp16(d, kp + off, on); pa_cp16(d + 2 * PA_BLOCK, vp + off, on);
            }
        }
        pa_commit();
    };
    look(0); load(0); look(1); load(1); look(2);
    PaTile<float, KV, D> t;
    if (mine < n_rows) t.start(a, s, kvh, mine, n_rows);
    for (int i = 0; i < n_stage; ++i) {
        pa_wait<1>();
        __syncthreads();                                  // the stage is here, and nobody reads the one before it
        load(i + 2);
        look(i + 3);
#pragma unroll 1
        for (int u = 0; u < 2; ++u) {
            const int key0 = i * STAGE + u * KEYS;
            if (key0 >= my_k1) break;
            const uint32_t kb = ring + i % 3 * BYTES + u * PA_BLOCK, vb = kb + 2 * PA_BLOCK;
            const bool edge = key0 + KEYS - 1 > t.first_last || key0 + KEYS > my_k1;
            t.scores(kb);
            t.weights(key0, my_k1, edge);
            t.values(smem, vb, key0, my_k1, edge);
        }
    }
    pa_wait<0>();
    if (mine >= n_rows) return;
    t.finish();
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int row = mine + (lane >> 2) + 8 * u;
        if (row >= n_rows) continue;
        const float l = u ? t.lb : t.la, inv = l == 0.0f ? 0.0f : 1.0f / l;
        const int tok = row / a.group, h = kvh * a.group + row % a.group;
        float * dst = (float *) (a.dst + (s.tok0 + tok) * a.nb_dst_tok + h * a.nb_dst_head) + (lane & 3) * 2;
#pragma unroll
        for (int c = 0; c < NC; ++c) *(float2 *) (dst + c * 8) = make_float2(t.o[c][2 * u] * inv, t.o[c][2 * u + 1] * inv);
        if (a.lse && (lane & 3) == 0) a.lse[(s.tok0 + tok) * a.n_head + h] = l == 0.0f ? -INFINITY : (u ? t.mb : t.ma) * 0.69314718f + logf(l);
    }
}

// Joins the partial items: one warp per row of a sequence.  An item's rounds lie in CTAs c0 .. c1 of the line; the first left its part in
// slot 1, the others in slot 0.
template <typename Q, int D>
__global__ void __launch_bounds__(128)
k_paged_join(const __grid_constant__ PaArgs a) {
    constexpr int DL = D / 32, ROUND = PA_BLOCK / (2 * D) * PA_WARPS;
    chain_release();
    chain_wait();
    const int lane = threadIdx.x & 31, seq = blockIdx.y, failed = pa_failed(a);
    const PaSeq s = pa_seq(a, seq);
    if (s.n_new == 0 || failed) return;
    const PaLine l = pa_line(a, ROUND, 0, seq, nullptr, nullptr);
    const int rounds = max(1, (s.len + ROUND - 1) / ROUND), tiles = (s.n_new * a.group + PA_ROWS - 1) / PA_ROWS;
    for (int64_t w = (int64_t) blockIdx.x * 4 + (threadIdx.x >> 5); w < (int64_t) s.n_new * a.n_head; w += (int64_t) gridDim.x * 4) {
        const int t = (int) (w / a.n_head), h = (int) (w - (int64_t) t * a.n_head), kvh = h / a.group, row = t * a.group + h % a.group;
        const int64_t p0 = l.before + ((int64_t) kvh * tiles + row / PA_ROWS) * (rounds + PA_START) + PA_START;      // its first round
        const int64_t c0 = ((p0 + 1) * a.stream - 1) / l.total, c1 = ((p0 + rounds) * a.stream - 1) / l.total;      // CTA c: from c * total / stream on
        if (c0 == c1) continue;
        const int n = (int) (c1 - c0 + 1);
        auto part = [&](int i) { return a.part + (((c0 + i) * 2 + (i == 0)) * PA_ROWS + row % PA_ROWS) * (D + 4); };
        float mx = -INFINITY;
        auto some = [&](int i) { return (c0 + i + 1) * l.total / a.stream > (c0 + i) * l.total / a.stream; };       // fewer rounds than CTAs leave some without
        for (int i = lane; i < n; i += 32) if (some(i)) mx = fmaxf(mx, part(i)[D]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float base = mx == -INFINITY ? 0.0f : mx;
        float sum = 0.0f, acc[DL] = {};
#pragma unroll 4
        for (int i = 0; i < n; ++i) {
            if (l.total < a.stream && !some(i)) continue;
            const float * p = part(i);
            const float f = pa_exp2(p[D] - base);
            sum += f * p[D + 1];                          // NaN of a part without a finite maximum stays NaN
#pragma unroll
            for (int j = 0; j < DL; ++j) acc[j] += f * p[lane * DL + j];
        }
        const int64_t out = (s.tok0 + t) * a.n_head + h;
#pragma unroll
        for (int j = 0; j < DL; ++j)
            ((Q *) (a.dst + (s.tok0 + t) * a.nb_dst_tok + h * a.nb_dst_head))[lane * DL + j] = (Q) (sum == 0.0f ? 0.0f : acc[j] / sum);
        if (a.lse && lane == 0) a.lse[out] = sum == 0.0f ? -INFINITY : mx * 0.69314718f + logf(sum);
    }
}

// Joins the splits of the tcgen05 form's last items: a warp a row, block (item, y).
template <typename Q, int D>
__global__ void __launch_bounds__(128)
k_paged_join_tc(const __grid_constant__ PaArgs a) {
    chain_release();
    chain_wait();
    constexpr int DL = D / 32;
    const int lane = threadIdx.x & 31, failed = pa_failed(a);
    const PaItem item = pa_item(a, a.n_whole + blockIdx.x * a.n_split);
    const PaSeq s = pa_seq(a, item.seq);
    const int row0 = item.tile * a.tile_rows, rows = min(a.tile_rows, s.n_new * a.group - row0);
    if (rows <= 0 || failed) return;
    const int n = min(a.n_split, max(1, (pa_reach(a, s, row0) + a.chunk - 1) / a.chunk));
    const int64_t step = (int64_t) a.tile_rows * (D + 4);
    for (int r = blockIdx.y * 4 + (threadIdx.x >> 5); r < rows; r += gridDim.y * 4) {
        const float * p = a.part + (item.slot * a.tile_rows + r) * (D + 4);
        float mx = -INFINITY;
        for (int i = lane; i < n; i += 32) mx = fmaxf(mx, p[i * step + D]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float base = mx == -INFINITY ? 0.0f : mx;
        float sum = 0.0f, acc[DL] = {};
#pragma unroll 4
        for (int i = 0; i < n; ++i) {
            const float f = pa_exp2(p[i * step + D] - base);
            sum += f * p[i * step + D + 1];               // NaN of a split without a finite maximum stays NaN
#pragma unroll
            for (int j = 0; j < DL; ++j) acc[j] += f * p[i * step + lane * DL + j];
        }
        const int t = (row0 + r) / a.group, h = item.kvh * a.group + (row0 + r) % a.group;
        const int64_t out = (s.tok0 + t) * a.n_head + h;
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
    if ((a->max_new < a->n_tok ? a->max_new : a->n_tok) >= (1ll << 30) || a->table_stride >= (1ll << 31)) return false;      // positions are 32 bits
    if (!a->tables || a->table_stride < 1 || !a->lens || !a->q_start || ((uintptr_t) a->tables | (uintptr_t) a->lens | (uintptr_t) a->q_start | (uintptr_t) a->lse | (uintptr_t) a->status) % 4) return false;
    if (!a->k_new != !a->v_new || (!attn && !a->k_new)) return false;
    const int64_t size = a->q_type == B200_TYPE_F32 ? 4 : 2, row = size * p->head_dim;
    if (a->k_new && (((uintptr_t) a->k_new | (uintptr_t) a->v_new | (uintptr_t) a->nb_new_tok | (uintptr_t) a->nb_new_head) % 16 ||
                     a->nb_new_tok < 0 || a->nb_new_head < 0)) return false;
    if (!attn) return true;
    if (!a->q || !a->dst || a->n_head < 1 || a->n_head % p->n_head_kv || a->n_head > 4096) return false;
    if ((a->max_new < a->n_tok ? a->max_new : a->n_tok) * (a->n_head / p->n_head_kv) >= (1ll << 30)) return false;
    if (((uintptr_t) a->q | (uintptr_t) a->dst | (uintptr_t) a->nb_q_tok | (uintptr_t) a->nb_q_head | (uintptr_t) a->nb_dst_tok | (uintptr_t) a->nb_dst_head) % 16) return false;
    if (a->nb_q_tok < 0 || a->nb_q_head < 0 || (a->n_head > 1 && a->nb_dst_head < row) || (a->n_tok > 1 && a->nb_dst_tok < row)) return false;
    const float log2 = a->scale * 1.44269504f;
    return log2 - log2 == 0.0f;                                        // finite
}

// Which kernel, and how its work is dealt out.
struct PaPlan { bool tc, wide, store; int stream, tiles, n_whole, n_split, chunk; int64_t items; };
static PaPlan pa_plan(const b200_page_pool * p, const b200_paged_attn_args * a) {
    PaPlan r = {};
    const int64_t group = a->n_head / p->n_head_kv;
    const int64_t new_max = a->max_new < a->n_tok ? a->max_new : a->n_tok, rows = new_max * group;
    // tcgen05 where its tiles of 128 or 256 rows are not mostly empty and the work fills the device, by the number of tiles of 16 rows and by them
    // times keys.  us, mma.sync and tcgen05, head_dim 64: 4 prompts of 256 tokens of 20 heads (1280 tiles) 24.5, 19.0; a chunk of 256 over 2256 keys
    // (320 tiles, 720k) 46, 38; but 1 prompt of 256 (320 tiles, 82k) 12.5, 15.9; a chunk of 256 over 8256 keys of 6 heads (96 tiles) 42, 57.
    // head_dim 128, 8 heads: 64 prompts of 128 rows (4096 tiles) 63, 45; a chunk of 64 rows over 8k keys (32 tiles, 258k) 38, 28; but 64
    // prompts of 48 rows (1536 tiles, 18k) 34, 41.  With up to 32 rows equal sequences gain a little, ragged ones lose more (16 of up to 32
    // tokens, 20 heads, up to 2500 keys: 51, 69).
    const int64_t small = (rows + PA_ROWS - 1) / PA_ROWS * p->n_head_kv * a->n_seq, work = small * a->max_len;
    r.tc = a->q_type != B200_TYPE_F32 && rows > 2 * PA_ROWS &&
           (p->head_dim == 64 ? small >= 640 || (small >= 160 && work >= 500000) : (small >= 512 && rows >= 128) || work >= 250000);
    const int64_t tile = r.tc ? PA_TC_ROWS(p->head_dim) : PA_ROWS, tiles = (rows + tile - 1) / tile;
    const int64_t round = r.tc ? PA_TC_KEYS(p->head_dim) : PA_BLOCK / (2 * p->head_dim) * PA_WARPS, rounds = (a->max_len + round - 1) / round;
    const int64_t resident = 148 * (r.tc ? PA_TC_CTAS(p->head_dim) : a->q_type == B200_TYPE_F32 ? 2 : 3);
    r.items = tiles * p->n_head_kv * a->n_seq;
    r.tiles = (int) tiles;
    r.wide = a->q_type == B200_TYPE_F32 && rows > PA_WIDE_MIN_ROWS && r.items >= PA_WIDE_MIN_ITEMS;
    r.store = a->k_new && (r.tc || r.wide || new_max > PA_ROWS);       // few new rows are stored by the kernel itself
    if (r.wide) return r;
    if (!r.tc) {
        // The line where items are long, or, from 12 rounds on, where they would leave the last wave half empty; many tiles of a chunk fill the
        // device by themselves (their reach differs, which the line does not know).  Single tokens, us without and with the line:
        // head_dim 64, 20 heads, 16 rounds (2000 keys): 1 sequence 15.9, 16.1; 4: 16.3, 19.9; 16: 36, 41.  head_dim 128, 8 heads, 16 rounds (1000
        // keys): 1 sequence 16.1, 16.9; 16: 17, 23; 64 (1.15 waves) 66, 57; 21 rounds: 1 sequence 19.9, 17.4; 64 92, 75.
        const bool tail = r.items > resident && r.items % resident <= resident / 2;
        if ((rounds >= 18 || (rounds >= 12 && tail)) && (tiles == 1 || r.items < 2 * resident)) {
            const int64_t want = r.items * rounds / 4;
            r.stream = (int) (want < resident ? want : resident);
        }
        return r;
    }
    const int64_t whole = r.items / resident * resident, rest = r.items - whole;
    int64_t split = rest ? resident / rest : 1;
    if (split > rounds / 4) split = rounds / 4;
    // The last of many waves is not worth the join; with four CTAs an SM no last wave is (64 chunks of 300 over 1300 keys, 20 heads: 338 us whole,
    // 370 split).  head_dim 128: 2 chunks of 2048 over 16k keys, 3.5 waves, 949 split, 1040 whole.
    if (split < 1 || whole > (p->head_dim == 64 ? 0 : 8 * resident)) split = 1;
    r.n_whole = (int) (split == 1 ? r.items : whole);
    r.chunk = split == 1 ? 0 : (int) ((rounds + split - 1) / split * round);
    r.n_split = split == 1 ? 1 : (int) ((a->max_len + r.chunk - 1) / r.chunk);
    return r;
}

extern "C" int64_t b200_paged_attn_workspace(const b200_page_pool * pool, const b200_paged_attn_args * a) {
    if (!a || !b200_pool_ok(pool, true) || a->n_tok < 1 || a->n_seq < 1 || a->max_new < 1 || a->max_len < 0 || a->max_len >= (1ll << 30) ||
        a->n_head < 1 || a->n_head % pool->n_head_kv) return 0;
    const PaPlan r = pa_plan(pool, a);
    // bounded, although not monotone in the sizes: split items have 148 (head_dim 128) or 592 (64) parts in all at most, the line has 444 CTAs: 20.6 MB
    return (r.tc ? (r.items - r.n_whole) * r.n_split * PA_TC_ROWS(pool->head_dim) : (int64_t) r.stream * 2 * PA_ROWS) * (pool->head_dim + 4) * 4;
}

static PaArgs pa_pack(const b200_page_pool * p, const b200_paged_attn_args * a) {
    PaArgs k = {};
    k.q = (const char *) a->q; k.nb_q_tok = a->nb_q_tok; k.nb_q_head = a->nb_q_head;
    k.dst = (char *) a->dst; k.nb_dst_tok = a->nb_dst_tok; k.nb_dst_head = a->nb_dst_head;
    k.k = (const char *) p->k + a->layer * p->nb_layer; k.v = (const char *) p->v + a->layer * p->nb_layer;
    k.nb_page = p->nb_page; k.nb_tok = p->nb_tok; k.nb_head = p->nb_head;
    k.tables = a->tables; k.table_stride = a->table_stride; k.lens = a->lens; k.q_start = a->q_start; k.status = a->status;
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
    int64_t n = (k.max_new + 7) / 8;
    const int64_t most = (148 * 8 + a->n_seq - 1) / a->n_seq;
    if (n > most) n = most;
    const bool f32 = a->q_type == B200_TYPE_F32, h = pool->type == B200_TYPE_F16;
    auto f = h ? (f32 ? k_paged_store<__half, true> : k_paged_store<__half, false>) : (f32 ? k_paged_store<__nv_bfloat16, true> : k_paged_store<__nv_bfloat16, false>);
    const cudaError_t e = launch_chained(f, dim3((unsigned) n, (unsigned) a->n_seq), dim3(256), 0, as_stream(stream), k, x, pool->head_dim == 64 ? 3 : 4);
    if (e != cudaSuccess) return (int) e;
    B200_RETURN_LAST();
}

template <typename Q, typename KV, int D>
static cudaError_t pa_launch(PaArgs & k, const PaNew & x, int n_seq, int64_t n_items, cudaStream_t st) {
    cudaError_t e;
    if constexpr (std::is_same<Q, KV>::value) {            // (f32 queries never go there)
        if (k.tile_rows != PA_ROWS) {
            e = pa_tc_launch(k, D, std::is_same<KV, __half>::value ? B200_TYPE_F16 : B200_TYPE_BF16, n_items, st);
            if (e != cudaSuccess || k.n_split == 1) return e;
            e = launch_chained(k_paged_join_tc<Q, D>, dim3((unsigned) (n_items - k.n_whole), (unsigned) k.tile_rows / 16), dim3(128), 0, st, k);
            if (e == cudaSuccess) B200_LAUNCHED();
            return e;
        }
    }
    const int64_t tiles = ((int64_t) k.max_new * k.group + PA_ROWS - 1) / PA_ROWS;
    const dim3 grid = k.stream ? dim3((unsigned) k.stream) : dim3((unsigned) tiles, (unsigned) k.n_head_kv, (unsigned) n_seq);
    // few items, one CTA per SM at most: eight warps share an item's blocks (5 beams of 20 heads, 431 keys, f32: 11.2 -> 8.8 us)
    if (!k.stream && n_items <= 148) {
        e = allow_once<k_paged_attn<Q, KV, D, 8>>(4 * 8 * PA_BLOCK);
        if (e == cudaSuccess) e = launch_chained(k_paged_attn<Q, KV, D, 8>, grid, dim3(256), 4 * 8 * PA_BLOCK, st, k, x);
    } else {
        e = allow_once<k_paged_attn<Q, KV, D, PA_WARPS>>(4 * PA_WARPS * PA_BLOCK);
        if (e == cudaSuccess) e = launch_chained(k_paged_attn<Q, KV, D, PA_WARPS>, grid, dim3(32 * PA_WARPS), 4 * PA_WARPS * PA_BLOCK, st, k, x);
    }
    if (e != cudaSuccess) return e;
    B200_LAUNCHED();
    if (!k.stream) return cudaGetLastError();
    const int64_t rows = (int64_t) k.max_new * k.n_head;
    e = launch_chained(k_paged_join<Q, D>, dim3((unsigned) (rows < 16384 ? (rows + 3) / 4 : 4096), (unsigned) n_seq), dim3(128), 0, st, k);
    if (e == cudaSuccess) B200_LAUNCHED();
    return e;
}

extern "C" int b200_paged_attn(const b200_page_pool * pool, const b200_paged_attn_args * a, void * stream) {
    if (!pa_args_ok(pool, a, true)) return B200_ERR_ARG;
    if (a->n_seq == 0 || a->n_tok == 0 || a->max_new == 0) return 0;
    PaArgs k = pa_pack(pool, a);
    const PaPlan r = pa_plan(pool, a);
    k.n_split = r.n_split; k.chunk = r.chunk; k.stream = r.stream; k.tile_rows = r.tc ? PA_TC_ROWS(pool->head_dim) : PA_ROWS; k.n_seq = a->n_seq;
    k.tiles = r.tiles; k.n_whole = r.n_whole;
    if (r.items > 0x7fffffff || (r.items - r.n_whole) * r.n_split > 0x7fffffff - r.n_whole) return B200_ERR_ARG;
    const int64_t need = b200_paged_attn_workspace(pool, a);
    if (need && (!a->workspace || (uintptr_t) a->workspace % 16 || a->workspace_bytes < need)) return B200_ERR_ARG;
    if (r.store) {
        const int rc = b200_paged_store(pool, a, stream);
        if (rc) return rc;
        k.early = 1;
    }
    const cudaStream_t st = as_stream(stream);
    const bool f32 = a->q_type == B200_TYPE_F32, h = pool->type == B200_TYPE_F16;
    const PaNew x = { r.store ? nullptr : (const char *) a->k_new, (const char *) a->v_new, a->nb_new_tok, a->nb_new_head };
    cudaError_t e;
    if (r.wide) {
        const dim3 grid((unsigned) ((k.max_new * (int64_t) k.group + PA_ROWS * PA_WIDE - 1) / (PA_ROWS * PA_WIDE)), (unsigned) k.n_head_kv, (unsigned) a->n_seq);
        auto f = pool->head_dim == 64 ? (h ? k_paged_attn_wide<__half, 64> : k_paged_attn_wide<__nv_bfloat16, 64>) : (h ? k_paged_attn_wide<__half, 128> : k_paged_attn_wide<__nv_bfloat16, 128>);
        e = launch_chained(f, grid, dim3(32 * PA_WIDE), 3 * 4 * PA_BLOCK, st, k);
        if (e != cudaSuccess) return (int) e;
        B200_RETURN_LAST();
    }
    if (pool->head_dim == 64)
        e = f32 ? (h ? pa_launch<float, __half, 64>(k, x, a->n_seq, r.items, st) : pa_launch<float, __nv_bfloat16, 64>(k, x, a->n_seq, r.items, st))
                : (h ? pa_launch<__half, __half, 64>(k, x, a->n_seq, r.items, st) : pa_launch<__nv_bfloat16, __nv_bfloat16, 64>(k, x, a->n_seq, r.items, st));
    else
        e = f32 ? (h ? pa_launch<float, __half, 128>(k, x, a->n_seq, r.items, st) : pa_launch<float, __nv_bfloat16, 128>(k, x, a->n_seq, r.items, st))
                : (h ? pa_launch<__half, __half, 128>(k, x, a->n_seq, r.items, st) : pa_launch<__nv_bfloat16, __nv_bfloat16, 128>(k, x, a->n_seq, r.items, st));
    return (int) e;
}
