// Beam search on the device: the next beams over (beam, vocabulary) and the reordering of per-beam state.
// Counterpart on the host in the reference: whisper_sample_token_topk and the candidate sort of whisper_full_with_state
// (src/whisper.cpp:5230-5430, 5880-6010), which scan and copy on the CPU.
#include "b200_common.cuh"
#include <cuda_bf16.h>

// ---- selection -----------------------------------------------------------------------------------
// score(b, v) = score[b] + (x - m) - log(sum exp(x - m)).  Within a row the order of the candidates is the order of the
// logits, so a row's n_beam best logits are all it can contribute: pass 1 cuts every row into slices and leaves, per slice,
// its maximum, its sum of exponentials and its n_beam best logits; pass 2 joins the slices of a sequence's rows and picks
// the n_beam best of their sorted lists.  The logits are read once and stay in registers.  With the slice in 8 (or 32) groups, the n_beam-th
// best of the groups' maxima bounds the slice's n_beam best from below, and about 7 logits reach it (5 beams, 8 groups: 8/8 + 8/7 + .. + 8/4):
// only those are looked at one by one.  Where equal logits make them more than SEL_CAP, the bound is taken once more over the threads' maxima
// with the index as the second part of the key; then the n_beam threads that reach it hold all that do.
// 320 rows of 51866 (f32): 65 us with a sorted list per warp, filled tile by tile; 35 with the n_beam best thread maxima of every warp as the
// bound and slices of four tiles (two CTAs an SM), 27 with two tiles (four CTAs), 23 with the groups' maxima.  No faster: CTAs of 128 threads (22.8),
// CTAs that stay and ask for their next slice ahead (37: what counts is how many slices are under way).
#define SEL_THREADS 256
#define SEL_EPT     16                              // logits per thread and tile
#define SEL_TILE    (SEL_THREADS * SEL_EPT)
#define SEL_MANY    2                               // tiles of a slice where rows are many (32 logits per thread); one tile otherwise
#define SEL_CAP     (B200_BEAM_MAX * SEL_EPT * SEL_MANY)
#define SEL_LISTS   32768                           // slices of a sequence's rows that pass 2 can join (a byte of shared memory each)

// order-preserving map of a float to an unsigned integer (larger float -> larger integer); 0 is left for "nothing"
__device__ __forceinline__ uint32_t sel_key(float x) {
    const uint32_t u = __float_as_uint(x);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float sel_val(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }
__device__ __forceinline__ unsigned long long sel_key(double x) {
    const unsigned long long u = (unsigned long long) __double_as_longlong(x);
    return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}
__device__ __forceinline__ double sel_val(unsigned long long k) {
    return __longlong_as_double((long long) ((k >> 63) ? (k & 0x7fffffffffffffffull) : ~k));
}
__device__ __forceinline__ unsigned long long sel_max(uint32_t hi, uint32_t lo) {        // over the warp
    const uint32_t h = __reduce_max_sync(0xffffffffu, hi);
    return (unsigned long long) h << 32 | __reduce_max_sync(0xffffffffu, hi == h ? lo : 0u);
}

// 2^x; below 2^-126 it is 0 (the plain form spends four more instructions on those)
__device__ __forceinline__ float sel_exp2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

// 16 consecutive bytes of logits with the widest loads that the row's alignment allows.  Which lane sums which logits does not depend
// on the alignment, so equal rows give equal bits wherever they lie.
template <typename T>
__device__ __forceinline__ uint4 sel_load(const T * p, int align) {
    union { uint4 q; uint2 h[2]; uint32_t w[4]; T t[16 / sizeof(T)]; } u;
    if (align >= 16)      u.q = *(const uint4 *) p;
    else if (align == 8)  { u.h[0] = ((const uint2 *) p)[0]; u.h[1] = ((const uint2 *) p)[1]; }
    else if (align == 4)  { for (int i = 0; i < 4; ++i) u.w[i] = ((const uint32_t *) p)[i]; }
    else                  { for (int i = 0; i < 16 / (int) sizeof(T); ++i) u.t[i] = p[i]; }
    return u.q;
}
template <typename T> __device__ __forceinline__ float sel_get(uint4 q, int i) { union { uint4 q; T t[16 / sizeof(T)]; } u; u.q = q; return (float) u.t[i]; }

struct SelSlices {            // workspace of a call: [rows][n_slice] maxima and sums, [rows][n_slice][n_beam] best logits
    float * m; double * s; float * x; int32_t * v;
};

// tiles of a slice: single tiles as long as larger slices would not fill the device twice (rows of 51866 f32 logits, us with one and two tiles: 5 rows
// 7.9, 8.3; 40 rows 9.7, 10.1; 60 rows 11.5, 11.0; 320 rows 28.3, 24.0)
static inline int sel_tiles(int64_t rows, int n_beam, int64_t n_vocab) {
    const int64_t slices = (n_vocab + SEL_TILE * SEL_MANY - 1) / (SEL_TILE * SEL_MANY);
    return rows * slices >= 148 * 2 || n_beam * ((n_vocab + SEL_TILE - 1) / SEL_TILE) > 4096 ? SEL_MANY : 1;
}
static inline int64_t sel_slices(int64_t rows, int n_beam, int64_t n_vocab) {
    const int64_t size = SEL_TILE * sel_tiles(rows, n_beam, n_vocab);
    return (n_vocab + size - 1) / size;
}

static inline SelSlices sel_layout(void * ws, int64_t rows, int64_t n_slice, int n_beam, int64_t * bytes) {
    const int64_t n = rows * n_slice;
    SelSlices p;
    char * b = (char *) ws;
    p.s = (double *) b;            b += 8 * n;
    p.m = (float *) b;             b += 4 * n;
    p.x = (float *) b;             b += 4 * n * n_beam;
    p.v = (int32_t *) b;           b += 4 * n * n_beam;
    *bytes = b - (char *) ws;
    return p;
}

template <typename T, int NT>
__global__ void __launch_bounds__(SEL_THREADS, 4)
k_beam_scan(const char * logits, int64_t nb_row, int n_vocab, const float * score, const uint8_t * done,
            const uint32_t * banned, int64_t banned_stride, int n_beam, SelSlices out) {
    constexpr int VEC = 16 / sizeof(T), NV = NT * SEL_EPT / VEC, NW = SEL_THREADS / 32;
    __shared__ double s_s[NW];
    __shared__ float s_grp[32];
    __shared__ unsigned long long s_top[NW * B200_BEAM_MAX], s_bound;
    __shared__ unsigned long long s_cand[SEL_CAP];
    __shared__ int s_n;
    chain_release();
    chain_wait();
    const int64_t row = blockIdx.x;
    const int slice = blockIdx.y, n_slice = gridDim.y, base = slice * SEL_TILE * NT;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const T * x_row = (const T *) (logits + row * nb_row);
    const int align = (uintptr_t) x_row & 15 ? (int) ((uintptr_t) x_row & (~(uintptr_t) x_row + 1)) : 16;      // 2, 4, 8 or 16
    const float sc = score[row];
    const uint8_t dn = done ? done[row] : 0;
    auto first = [&](int j) { return base + (j * SEL_THREADS + tid) * VEC; };
    float x[NV][VEC];
    if (n_vocab - base >= SEL_TILE * NT) {
        uint4 raw[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) raw[j] = sel_load<T>(x_row + first(j), align);
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) x[j][i] = fmaxf(sel_get<T>(raw[j], i), -INFINITY);      // no NaN
    } else {                                    // the row ends in this slice
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int e = first(j);
            uint4 raw;
            if (e + VEC <= n_vocab) raw = sel_load<T>(x_row + e, align);
            else {
                union { uint4 q; T t[VEC]; } u;
#pragma unroll
                for (int i = 0; i < VEC; ++i) u.t[i] = (T) (e + i < n_vocab ? (float) x_row[e + i] : -INFINITY);
                raw = u.q;
            }
#pragma unroll
            for (int i = 0; i < VEC; ++i) x[j][i] = fmaxf(sel_get<T>(raw, i), -INFINITY);
        }
    }
    if (!(sc > -INFINITY) || dn) return;
    if (banned) {
        const uint32_t * mask = banned + row * banned_stride;
        uint32_t w[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) w[j] = first(j) < n_vocab ? mask[first(j) >> 5] >> (first(j) & 31) : 0;      // VEC divides 32 and first(j) is a multiple of it
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) if (w[j] & (1u << i)) x[j][i] = -INFINITY;
    }
    if (sc == INFINITY) {                        // the score of all of them: equal candidates, of which the lowest tokens count, not the largest logits
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) if (fabsf(x[j][i]) < INFINITY) x[j][i] = 0.0f;
    }
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) m = fmaxf(m, x[j][i]);
    // groups: the warps, or eight lanes each
    const int n_grp = n_beam <= NW ? NW : 32;
    float g = m;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
    if (n_beam <= NW) {
        g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, 8));
        g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, 16));
        if (lane == 0) s_grp[warp] = g;
    } else if ((lane & 7) == 0) s_grp[warp * 4 + (lane >> 3)] = g;
    if (tid == 0) s_n = 0;
    __syncthreads();
    // every warp: the best group, and the n_beam-th best
    const float mine = lane < n_grp ? s_grp[lane] : -INFINITY;
    float mx = mine;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const int64_t at = row * n_slice + slice;
    if (mx == -INFINITY) {
        if (tid == 0) { out.m[at] = -INFINITY; out.s[at] = 0.0; }
        if (tid < n_beam) out.v[at * n_beam + tid] = -1;
        return;
    }
    int rank = 0;
    for (int o = 0; o < n_grp; ++o) { const float v = __shfl_sync(0xffffffffu, mine, o); rank += v > mine || (v == mine && o < lane); }
    const unsigned who = __ballot_sync(0xffffffffu, lane < n_grp && rank == n_beam - 1);
    const float bar = __shfl_sync(0xffffffffu, mine, __ffs(who) - 1);
    // sum of exp(x - mx): f32 within a thread, joined in f64
    float se = 0.0f;
    if (mx < INFINITY) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) se += sel_exp2((x[j][i] - mx) * 1.44269504f);
    } else {                                     // infinite logits share the row
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) se += x[j][i] == INFINITY ? 1.0f : 0.0f;
    }
    double sd = se;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sd += __shfl_xor_sync(0xffffffffu, sd, o);
    if (lane == 0) s_s[warp] = sd;
    __syncthreads();
    auto key = [&](int j, int i) { return (unsigned long long) sel_key(x[j][i] + 0.0f) << 32 | ~(uint32_t) (first(j) + i); };      // one zero
    if (m >= bar && m > -INFINITY) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float v = x[j][0];
#pragma unroll
            for (int i = 1; i < VEC; ++i) v = fmaxf(v, x[j][i]);
            if (v >= bar && v > -INFINITY) {
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    if (x[j][i] >= bar && x[j][i] > -INFINITY) {
                        const int c = atomicAdd(&s_n, 1);
                        if (c < SEL_CAP) s_cand[c] = key(j, i);      // the order of arrival does not matter: they are ranked
                    }
            }
        }
    }
    __syncthreads();
    if (s_n > SEL_CAP) {                         // equal logits: once more with unique keys, over the n_beam best thread maxima of every warp
        unsigned long long k = 0;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) if (k == 0 && x[j][i] == m && m > -INFINITY) k = key(j, i);      // the lowest index: indices ascend
        unsigned long long left = k;
        for (int r = 0; r < n_beam; ++r) {
            const unsigned long long top = sel_max((uint32_t) (left >> 32), (uint32_t) left);
            if (lane == 0) s_top[warp * n_beam + r] = top;
            if (left == top) left = 0;
        }
        __syncthreads();
        if (tid == 0) { s_n = 0; s_bound = 1; }  // fewer candidates than beams: all that there are
        __syncthreads();
        if (tid < NW * n_beam) {
            const unsigned long long t = s_top[tid];
            int above = 0;
            for (int o = 0; o < NW * n_beam; ++o) above += s_top[o] > t;
            if (t && above == n_beam - 1) s_bound = t;
        }
        __syncthreads();
        const unsigned long long bound = s_bound;
        if (k >= bound) {
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < VEC; ++i) if (x[j][i] > -INFINITY && key(j, i) >= bound) s_cand[atomicAdd(&s_n, 1)] = key(j, i);
        }
        __syncthreads();
    }
    const int n = s_n;
    for (int c = tid; c < n; c += SEL_THREADS) {
        const unsigned long long k = s_cand[c];
        int rank = 0;
        for (int o = 0; o < n; ++o) rank += s_cand[o] > k;
        if (rank < n_beam) {
            out.x[at * n_beam + rank] = sel_val((uint32_t) (k >> 32));
            out.v[at * n_beam + rank] = (int32_t) ~(uint32_t) k;
        }
    }
    if (tid >= n && tid < n_beam) out.v[at * n_beam + tid] = -1;
    if (tid == SEL_THREADS - 1) {
        double sum = s_s[0];
#pragma unroll
        for (int w = 1; w < NW; ++w) sum += s_s[w];
        out.m[at] = mx; out.s[at] = sum;
    }
}

// One CTA per sequence: a warp per beam forms the logarithm of its sum, then n_beam rounds of an arg-max pick the best candidates.  Keys are
// (score as ordered 64-bit integer, lowest beam * n_vocab + token).  Bound by latency: all candidates are loaded at once, before the sums are
// known, and stay in registers (FLAT, up to SEL_HELD per thread); only where they are more, a thread holds the heads of its slices' sorted
// lists (list l = beam * n_slice + slice belongs to thread l mod blockDim) and loads the next ones as they are taken.
#define SEL_HELD 4
template <bool FLAT>
__global__ void __launch_bounds__(1024)
k_beam_pick(SelSlices in, const float * score, const uint8_t * done, int n_beam, int n_slice, int n_vocab, int eos,
            float * score_out, int32_t * token_out, int32_t * parent_out, uint8_t * done_out) {
    chain_release();
    chain_wait();
    extern __shared__ unsigned char s_head[];              // next entry of every list
    __shared__ double s_score[B200_BEAM_MAX], s_m[B200_BEAM_MAX], s_log[B200_BEAM_MAX];
    __shared__ uint8_t s_done[B200_BEAM_MAX], s_live[B200_BEAM_MAX];
    __shared__ uint32_t s_hi[2][32], s_lo[2][32], s_ix[2][32];
    const int64_t row0 = (int64_t) blockIdx.x * n_beam;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n_warp = blockDim.x >> 5, n_list = n_beam * n_slice, per_beam = n_slice * n_beam;
    float held_x[SEL_HELD];
    int   held_v[SEL_HELD];
    if (FLAT) {
#pragma unroll
        for (int i = 0; i < SEL_HELD; ++i) {
            const int c = i * blockDim.x + tid;
            held_x[i] = 0.0f; held_v[i] = -1;
            if (c < n_list * n_beam) { held_x[i] = in.x[row0 * per_beam + c]; held_v[i] = in.v[row0 * per_beam + c]; }
        }
    }
    for (int b = warp; b < n_beam; b += n_warp) {
        const float sc = score[row0 + b];
        const bool d = done && done[row0 + b], ok = sc > -INFINITY, live = ok && !d;
        const float * bm = in.m + (row0 + b) * n_slice;
        const double * bs = in.s + (row0 + b) * n_slice;
        const float m0 = lane < n_slice ? bm[lane] : -INFINITY;             // (a row that is not live left nothing here: not used)
        const double s0 = lane < n_slice ? bs[lane] : 0.0;
        float m = m0;
        for (int j = lane + 32; j < n_slice; j += 32) m = fmaxf(m, bm[j]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        double s = m0 == m ? s0 : m0 > -INFINITY ? s0 * (double) __expf(m0 - m) : 0.0;
        for (int j = lane + 32; j < n_slice; j += 32) {
            const float mj = bm[j];
            s += mj == m ? bs[j] : mj > -INFINITY ? bs[j] * (double) __expf(mj - m) : 0.0;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) {
            s_score[b] = sc; s_m[b] = m; s_log[b] = live && m > -INFINITY ? log(s) : 0.0;
            s_done[b] = d; s_live[b] = live && m > -INFINITY ? 1 : ok && d ? 2 : 0;
        }
    }
    if (!FLAT) for (int l = tid; l < n_list; l += blockDim.x) s_head[l] = 0;
    __syncthreads();

    // key of the candidate (beam b, token, logit): 0 = none.  A done beam has one, in its first place
    auto value = [&](int b, bool first, int tok, float x, uint32_t & ix) -> unsigned long long {
        double v;
        if (s_live[b] == 1) {
            if (tok < 0) return 0;
            v = s_score[b] + ((x == s_m[b] ? 0.0 : (double) x - s_m[b]) - s_log[b]);
            if (!(v > -INFINITY)) return 0;
        } else if (s_live[b] == 2 && first) {
            tok = eos >= 0 && eos < n_vocab ? eos : 0;             // its place among equals; the token itself may be any number
            v = s_score[b];
        } else return 0;
        ix = ~(uint32_t) (b * n_vocab + tok);
        return sel_key(v + 0.0);                                   // one zero
    };
    unsigned long long keys[SEL_HELD] = {}, mine = 0;
    uint32_t ixs[SEL_HELD] = {}, mine_ix = 0;                       // ~(b * n_vocab + token)
    int mine_l = 0;
    if (FLAT) {
#pragma unroll
        for (int i = 0; i < SEL_HELD; ++i) {
            const int c = i * blockDim.x + tid;
            if (c < n_list * n_beam) { const int b = c / per_beam; keys[i] = value(b, c == b * per_beam, held_v[i], held_x[i], ixs[i]); }
        }
    }
    auto look = [&]() {                                            // best of what this thread holds
        mine = 0; mine_ix = 0;
        if (FLAT) {
#pragma unroll
            for (int i = 0; i < SEL_HELD; ++i)
                if (keys[i] > mine || (keys[i] == mine && ixs[i] > mine_ix)) { mine = keys[i]; mine_ix = ixs[i]; mine_l = i; }
        } else {
            for (int l = tid; l < n_list; l += blockDim.x) {
                const int b = l / n_slice, h = s_head[l];
                if (h >= n_beam) continue;
                const int64_t at = (row0 * n_slice + l) * n_beam + h;
                uint32_t ix = 0;
                const unsigned long long k = value(b, l == b * n_slice && h == 0, in.v[at], in.x[at], ix);
                if (k > mine || (k == mine && ix > mine_ix)) { mine = k; mine_ix = ix; mine_l = l; }
            }
        }
    };
    look();
    for (int r = 0; r < n_beam; ++r) {
        const uint32_t h = (uint32_t) (mine >> 32), l = (uint32_t) mine;
        uint32_t bh = __reduce_max_sync(0xffffffffu, h);
        uint32_t bl = __reduce_max_sync(0xffffffffu, h == bh ? l : 0u);
        uint32_t bi = __reduce_max_sync(0xffffffffu, h == bh && l == bl ? mine_ix : 0u);
        if (n_warp > 1) {
            if (lane == 0) { s_hi[r & 1][warp] = bh; s_lo[r & 1][warp] = bl; s_ix[r & 1][warp] = bi; }
            __syncthreads();
            const uint32_t wh = lane < n_warp ? s_hi[r & 1][lane] : 0, wl = lane < n_warp ? s_lo[r & 1][lane] : 0, wi = lane < n_warp ? s_ix[r & 1][lane] : 0;
            bh = __reduce_max_sync(0xffffffffu, wh);
            bl = __reduce_max_sync(0xffffffffu, wh == bh ? wl : 0u);
            bi = __reduce_max_sync(0xffffffffu, wh == bh && wl == bl ? wi : 0u);
        }
        const unsigned long long top = (unsigned long long) bh << 32 | bl;
        if (top != 0 && mine == top && mine_ix == bi) {
            const uint32_t flat = ~bi;
            const int b = (int) (flat / (uint32_t) n_vocab), tok = s_live[b] == 2 ? eos : (int) (flat - (uint32_t) b * (uint32_t) n_vocab);
            score_out[row0 + r] = (float) sel_val(top);
            token_out[row0 + r] = tok;
            parent_out[row0 + r] = b;
            done_out[row0 + r] = s_done[b] || tok == eos;
            if (FLAT) {
#pragma unroll
                for (int i = 0; i < SEL_HELD; ++i) if (i == mine_l) { keys[i] = 0; ixs[i] = 0; }
            } else ++s_head[mine_l];
            look();
        }
        if (top == 0 && tid == 0) { score_out[row0 + r] = -INFINITY; token_out[row0 + r] = -1; parent_out[row0 + r] = -1; done_out[row0 + r] = 1; }
    }
}

static bool sel_sizes_ok(int n_seq, int n_beam, int64_t n_vocab) {
    return n_seq >= 0 && n_beam >= 1 && n_beam <= B200_BEAM_MAX && n_vocab >= 1 && n_vocab <= (1ll << 30) && n_vocab * n_beam < (1ll << 31) &&
           n_beam * ((n_vocab + SEL_TILE * SEL_MANY - 1) / (SEL_TILE * SEL_MANY)) <= SEL_LISTS && (int64_t) n_seq * n_beam <= 0x7fffffff;
}

extern "C" int64_t b200_beam_select_workspace(int n_seq, int n_beam, int64_t n_vocab) {
    if (!sel_sizes_ok(n_seq, n_beam, n_vocab)) return 0;
    int64_t bytes;
    const int64_t rows = (int64_t) n_seq * n_beam;
    sel_layout(nullptr, rows, sel_slices(rows, n_beam, n_vocab), n_beam, &bytes);
    return bytes;
}

extern "C" int b200_beam_select(const b200_beam_select_args * a, void * stream) {
    if (!a || !sel_sizes_ok(a->n_seq, a->n_beam, a->n_vocab)) return B200_ERR_ARG;
    const int64_t rows = (int64_t) a->n_seq * a->n_beam, n_slice = sel_slices(rows, a->n_beam, a->n_vocab);
    const int size = a->type == B200_TYPE_F32 ? 4 : a->type == B200_TYPE_F16 || a->type == B200_TYPE_BF16 ? 2 : 0;
    if (!size || a->nb_row % size || a->nb_row < a->n_vocab * size || a->banned_stride < 0) return B200_ERR_ARG;
    if (a->n_seq == 0) return 0;
    if (!a->logits || !a->score || !a->score_out || !a->token_out || !a->parent_out || !a->done_out || (uintptr_t) a->logits % size) return B200_ERR_ARG;
    if (((uintptr_t) a->score | (uintptr_t) a->banned | (uintptr_t) a->score_out | (uintptr_t) a->token_out | (uintptr_t) a->parent_out) % 4) return B200_ERR_ARG;
    if (!a->workspace || (uintptr_t) a->workspace % 16 || a->workspace_bytes < b200_beam_select_workspace(a->n_seq, a->n_beam, a->n_vocab)) return B200_ERR_ARG;
    int64_t bytes;
    const SelSlices ws = sel_layout(a->workspace, rows, n_slice, a->n_beam, &bytes);
    const cudaStream_t st = as_stream(stream);
    const dim3 grid((unsigned) rows, (unsigned) n_slice);
    const bool many = sel_tiles(rows, a->n_beam, a->n_vocab) > 1;
    auto scan = a->type == B200_TYPE_F32 ? (many ? k_beam_scan<float, SEL_MANY> : k_beam_scan<float, 1>)
              : a->type == B200_TYPE_F16 ? (many ? k_beam_scan<__half, SEL_MANY> : k_beam_scan<__half, 1>)
                                         : (many ? k_beam_scan<__nv_bfloat16, SEL_MANY> : k_beam_scan<__nv_bfloat16, 1>);
    cudaError_t e = launch_chained(scan, grid, dim3(SEL_THREADS), 0, st, (const char *) a->logits, a->nb_row, (int) a->n_vocab, a->score, a->done,
                                   a->banned, a->banned_stride, a->n_beam, ws);
    if (e != cudaSuccess) return (int) e;
    B200_LAUNCHED();
    const int64_t n_list = n_slice * a->n_beam, held = (n_list * a->n_beam + SEL_HELD - 1) / SEL_HELD;
    const bool flat = held <= 1024;
    int64_t lanes = flat ? held : n_list;
    if (lanes < 32 * a->n_beam) lanes = 32 * a->n_beam;
    const unsigned threads = (unsigned) (lanes >= 1024 ? 1024 : (lanes + 31) / 32 * 32);
    e = launch_chained(flat ? k_beam_pick<true> : k_beam_pick<false>, dim3((unsigned) a->n_seq), dim3(threads), flat ? 0 : (size_t) n_list, st, ws, a->score, a->done,
                       a->n_beam, (int) n_slice, (int) a->n_vocab, (int) a->eos, a->score_out, a->token_out, a->parent_out, a->done_out);
    if (e != cudaSuccess) return (int) e;
    B200_RETURN_LAST();
}

// ---- reordering ----------------------------------------------------------------------------------
// A thread owns one column (up to 16 bytes at the same offset of every row of a sequence): it loads the columns of all
// parents and only then stores, so the move is in place without a second buffer, and a beam that follows itself costs
// nothing.  Bound by memory: rows that change are written once, their parents read once (a parent of several beams comes
// from L1 the second time).  Up to 8 beams a thread has two columns, for more loads under way (40 rows of 1.1 MB in 64 outer steps: 661 us,
// 724 with one; 6.07 TB/s).
#define REORDER_THREADS 256
#define REORDER_BLOCKS  8
struct ReorderBlock { char * base; int64_t nb_outer, nb_row, row_bytes, first; unsigned tiles, n_outer; int vec; };
struct ReorderArgs { ReorderBlock b[REORDER_BLOCKS]; int n; };

// COLS columns of 16 bytes, `step` bytes apart, all of them inside the row
template <int NB, int COLS>
__device__ __forceinline__ void reorder_vectors(char * col, int64_t step, int64_t nb_row, const int (&p)[NB], int n_beam) {
    uint4 v[COLS][NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) if (b < n_beam && p[b] != b) {
#pragma unroll
        for (int c = 0; c < COLS; ++c) v[c][b] = *(const uint4 *) (col + c * step + p[b] * nb_row);
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) if (b < n_beam && p[b] != b) {
#pragma unroll
        for (int c = 0; c < COLS; ++c) *(uint4 *) (col + c * step + b * nb_row) = v[c][b];
    }
}
// `n` values of type V of one column, one after the other
template <typename V, int NB>
__device__ __forceinline__ void reorder_values(char * col, int64_t n, int64_t nb_row, const int (&p)[NB], int n_beam) {
    for (int64_t i = 0; i < n; ++i) {
        V v[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) if (b < n_beam && p[b] != b) v[b] = ((const V *) (col + p[b] * nb_row))[i];
#pragma unroll
        for (int b = 0; b < NB; ++b) if (b < n_beam && p[b] != b) ((V *) (col + b * nb_row))[i] = v[b];
    }
}

template <int NB> struct ReorderCols { static constexpr int n = NB <= 8 ? 2 : 1; };

template <int NB>
__global__ void __launch_bounds__(REORDER_THREADS)
k_beam_reorder(const __grid_constant__ ReorderArgs a, const int32_t * parent, int n_seq, int n_beam) {
    constexpr int COLS = ReorderCols<NB>::n;
    chain_release();
    chain_wait();
    int k = 0;
    while (k + 1 < a.n && (int64_t) blockIdx.x >= a.b[k + 1].first) ++k;
    const ReorderBlock & blk = a.b[k];
    int64_t r = (int64_t) blockIdx.x - blk.first;
    const unsigned tile = (unsigned) (r % blk.tiles); r /= blk.tiles;
    const int seq = (int) (r % n_seq);
    const int64_t outer = r / n_seq;
    int p[NB];
    bool any = false;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        p[b] = b;
        if (b < n_beam) {
            const int q = parent[(int64_t) seq * n_beam + b];
            if (q >= 0 && q < n_beam) p[b] = q;
            any |= p[b] != b;
        }
    }
    if (!any) return;
    const int64_t step = (int64_t) REORDER_THREADS * blk.vec, off = tile * COLS * step + threadIdx.x * blk.vec;
    char * col = blk.base + outer * blk.nb_outer + (int64_t) seq * n_beam * blk.nb_row + off;
    int64_t left = blk.row_bytes - off;
    if (blk.vec == 16 && left >= (COLS - 1) * step + 16) { reorder_vectors<NB, COLS>(col, step, blk.nb_row, p, n_beam); return; }
    for (int c = 0; c < COLS && left > 0; ++c, col += step, left -= step) {
        if (left >= blk.vec) {
            if (blk.vec == 16)     reorder_vectors<NB, 1>(col, 0, blk.nb_row, p, n_beam);
            else if (blk.vec == 4) reorder_values<uint32_t, NB>(col, 1, blk.nb_row, p, n_beam);
            else                   reorder_values<unsigned char, NB>(col, 1, blk.nb_row, p, n_beam);
        } else reorder_values<unsigned char, NB>(col, left, blk.nb_row, p, n_beam);      // the end of a row that is no multiple of the vector
    }
}

extern "C" int b200_beam_reorder(const b200_beam_block * blocks, int n_blocks, const int32_t * parent, int n_seq, int n_beam, void * stream) {
    if (n_blocks < 0 || n_blocks > REORDER_BLOCKS || n_seq < 0 || n_beam < 1 || n_beam > B200_BEAM_MAX || (n_blocks && !blocks)) return B200_ERR_ARG;
    ReorderArgs a = {};
    int64_t ctas = 0;
    for (int i = 0; i < n_blocks; ++i) {
        const b200_beam_block & s = blocks[i];
        if (s.n_outer < 0 || s.row_bytes < 0 || s.n_outer > 0x7fffffff || s.row_bytes > (1ll << 40)) return B200_ERR_ARG;
        if (s.n_outer == 0 || s.row_bytes == 0 || n_seq == 0 || n_beam == 1) continue;
        const int64_t rows = (int64_t) n_seq * n_beam;
        if (!s.base || s.nb_row < s.row_bytes || s.nb_row > (1ll << 40) / rows || s.nb_outer < 0 || s.nb_outer > (1ll << 50) / s.n_outer) return B200_ERR_ARG;
        if (s.n_outer > 1 && s.nb_outer < (rows - 1) * s.nb_row + s.row_bytes &&          // rows inside an outer step, or outer steps inside a row
            (s.nb_outer < s.row_bytes || s.nb_row < (s.n_outer - 1) * s.nb_outer + s.row_bytes)) return B200_ERR_ARG;
        const uintptr_t bits = (uintptr_t) s.base | (uintptr_t) s.nb_row | (s.n_outer > 1 ? (uintptr_t) s.nb_outer : 0);
        ReorderBlock & d = a.b[a.n++];
        d.base = (char *) s.base; d.nb_outer = s.nb_outer; d.nb_row = s.nb_row; d.row_bytes = s.row_bytes; d.first = ctas;
        d.vec = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1;
        d.n_outer = (unsigned) s.n_outer;
        const int64_t tile = (int64_t) d.vec * REORDER_THREADS * (n_beam <= 8 ? ReorderCols<8>::n : ReorderCols<16>::n), tiles = (s.row_bytes + tile - 1) / tile;
        if (tiles > 0x7fffffff) return B200_ERR_ARG;
        d.tiles = (unsigned) tiles;
        if (tiles * s.n_outer > 0x7fffffff || tiles * s.n_outer * n_seq > 0x7fffffff - ctas) return B200_ERR_ARG;
        ctas += tiles * s.n_outer * n_seq;
    }
    if (ctas == 0) return 0;
    if (!parent || (uintptr_t) parent % 4) return B200_ERR_ARG;
    auto k = n_beam <= 4 ? k_beam_reorder<4> : n_beam <= 8 ? k_beam_reorder<8> : n_beam <= 16 ? k_beam_reorder<16> : k_beam_reorder<32>;
    const cudaError_t e = launch_chained(k, dim3((unsigned) ctas), dim3(REORDER_THREADS), 0, as_stream(stream), a, parent, n_seq, n_beam);
    if (e != cudaSuccess) return (int) e;
    B200_RETURN_LAST();
}
