// Attention of many rows over a paged key/value cache on the fifth-generation tensor cores (tcgen05.mma, scores, weights and
// accumulators in tensor memory).  Operator and row numbering as in k_paged_attn.cu; 16-bit queries only.
//
// A CTA takes one or two tiles of 128 rows of one sequence and key/value head over one split of the keys, in blocks of BN keys:
//     S_t = Q_t K^T   (M 128, N BN, K head_dim)   both operands K-major in shared memory, 128-byte swizzle
//     O_t += P_t V    (M 128, N head_dim, K BN)   P_t from tensor memory (over S_t, 16-bit), V as stored: N-major, 128-byte swizzle
// While the softmax of one tile runs the tensor core has to have other work.  head_dim 128: two tiles in a CTA of 352 threads, which fill
// tensor memory (2 x (128 + 128) columns) and shared memory (192 KB), one CTA on an SM, BN = 128.  head_dim 64: one tile in a CTA of 224
// threads and four CTAs on an SM, BN = 64, so that short prompts do not leave half of a CTA's rows empty.
// Roles (NTILE tiles):
//   4 NTILE warps    softmax: a thread owns a row.  It reads its scores (tcgen05.ld), masks only blocks that some row does not see wholly,
//                    and writes the weights back as P.  The reference point of the exponentials is the running maximum, but it follows it
//                    only when the maximum has grown by more than 2^8: the weights stay below 256, the sums are exact in the same sense,
//                    and the rescaling of O (a read and a write of tensor memory) is rare.  f16 weights, which have all their bits only from
//                    2^-14 on, are 2^11 at the reference point and follow from 2^4 on (PtLag).  All exponentials go to the exponential unit:
//                    one of eight pairs as a polynomial on the FMA pipe made a chunk of 2048 over 16k keys slower (932 -> 966 us), one
//                    of four more so (1004 us).
//   1 warp           one thread issues all MMAs.  S_t(j+1) follows P_t V(j) in issue order, so the commit behind S_t(j+1) also says that
//                    O_t is at rest and that P_t may be overwritten; no further barrier is needed for either.
//   2 warps          bring K and V by TMA, page by page into the swizzled tile, where pages fit into blocks or blocks into pages (page
//                    sizes 8, 16, 32, .. and multiples of BN); otherwise per key one page lookup and 16-byte cp.async.  Zeros for keys
//                    out of reach and pages out of the pool.
// Measured, head_dim 128, bf16, chunks of 2048 queries over 16k keys, 32 heads on 8: 946 us, 1.09 PFLOP/s.  What bounds it is the chain of a
// tile: its softmax, then P V and the next Q K^T, while the other tile's softmax and products run beside it.  Tried without gain: P
// handed over in two halves (1097 against 1037 us), two score buffers with blocks of 64 keys (1661: Q K^T with N = 64 reads Q from shared
// memory twice as often), two threads a row (981 against 967).
// 0 * v is not 0 where v is infinite or NaN: in blocks that are not wholly seen the V warp takes such values out of its tile and raises
// a flag; the rows that do see them add them at the end, from the pages.
// All waits are bounded (about a second), record a code (b200_paged_attn_status) and make every role leave through the exit that frees
// tensor memory.
#include "paged_attn.cuh"
#include <cuda.h>
#include <string.h>

__device__ int g_pa_status;

extern "C" int b200_paged_attn_status(void) {
    static const int none = 0;
    int v = 0;
    cudaError_t e = cudaDeviceSynchronize();              // all streams: those that do not wait for the default stream as well
    if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&v, g_pa_status, sizeof(v));
    if (e == cudaSuccess && v != 0) e = cudaMemcpyToSymbol(g_pa_status, &none, sizeof(none));
    return e == cudaSuccess ? v : (int) e;
}

// powers of two: how far the maximum may run ahead of the reference point, the weight at the reference point; and the factor that takes the latter out
// (f16, 8 and 2^7 against 4 and 2^11: no difference in time on a chunk of 2048 over 16k keys, 16 times the step for the smallest weights; 8 and no raise is 1%
// faster, 1107 against 1118 us, and loses them)
template <typename T> struct PtLag { static constexpr float lag = 8.0f, raise = 0.0f, lower = 1.0f; };
template <> struct PtLag<__half> { static constexpr float lag = 4.0f, raise = 11.0f, lower = 1.0f / 2048.0f; };

#define PT_THREADS(NTILE) (128 * (NTILE) + 96)

template <int D, int BN, int NS, int NTILE> struct PtSmem {
    static constexpr int TILE = BN * D * 2, QT = 128 * D * 2;
    static constexpr int Q = 0, K = NTILE * QT, V = K + NS * TILE, BAR = V + NS * TILE;
    static constexpr int N_BAR = 5 * NS + 7;             // k_full, k_empty, v_full, v_empty, v_here [NS]; q_full; s_full, p_full, o_full [2]
    static constexpr int MISC = BAR + N_BAR * 8;         // tensor-memory address, abort flag, odd-value flag
    static constexpr int BYTES = MISC + 16 + 1024;       // the dynamic array starts on 16 bytes: tiles are moved to 1024
};

__device__ __forceinline__ bool pt_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// bounded wait: false after about a second, or when another role has given up; the clock is read only after many failed polls
__device__ __noinline__ bool pt_wait_slow(uint32_t bar, uint32_t parity, volatile int * abort_flag, int code) {
    unsigned long long t0 = 0, t;
    for (uint32_t i = 0; i < (1u << 28); ++i) {
        if (pt_try(bar, parity)) return true;
        if ((i & 255) == 255) {
            if (*abort_flag) return false;
            asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
            if (t0 == 0) t0 = t;
            else if (t - t0 > 1000000000ull) break;
        }
    }
    *abort_flag = 1;
    atomicCAS(&g_pa_status, 0, code);
    return false;
}
// up to 1024 polls in one piece of assembly
__device__ __forceinline__ bool pt_poll(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p, q;\n\t.reg .u32 i;\n\tmov.u32 i, 0;\n"
                 "poll_%=:\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t@p bra seen_%=;\n\tadd.u32 i, i, 1;\n\tsetp.lt.u32 q, i, 1024;\n\t@q bra poll_%=;\n"
                 "seen_%=:\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool pt_wait(uint32_t bar, uint32_t parity, volatile int * abort_flag, int code) {       // one thread
    return pt_poll(bar, parity) || pt_wait_slow(bar, parity, abort_flag, code);
}
// A warp waits with all its lanes and branches on a vote: with one lane polling for the others the warp stayed split afterwards and
// paid for every shuffle and .aligned instruction (a chunk of 2048 over 16k keys: 10.0 ms).
__device__ __forceinline__ bool pt_wait_warp(uint32_t bar, uint32_t parity, volatile int * abort_flag, int code) {
    bool ok = pt_try(bar, parity);
    if (!__all_sync(0xffffffffu, ok)) {
        ok = pt_poll(bar, parity);
        if (!__all_sync(0xffffffffu, ok)) {
            if (!ok) ok = pt_wait_slow(bar, parity, abort_flag, code);
            __syncwarp();
        }
    }
    return __all_sync(0xffffffffu, ok);
}
__device__ __forceinline__ void pt_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(bar) : "memory"); }
__device__ __forceinline__ void pt_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(bar) : "memory");
}
__device__ __forceinline__ void pt_proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void pt_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pt_after()  { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// shared-memory matrix descriptor, 128-byte swizzle (rows of 128 bytes, 8-row groups of 1024 bytes); lbo: bytes between 64-element
// columns of an N-major operand
__device__ __forceinline__ uint64_t pt_desc(uint32_t addr, uint32_t lbo) {
    return (uint64_t) ((addr >> 4) & 0x3fff) | (uint64_t) ((lbo >> 4) & 0x3fff) << 16 | (uint64_t) (1024 >> 4) << 32 | (uint64_t) 1 << 46 | (uint64_t) 2 << 61;
}
__device__ __forceinline__ void pt_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void pt_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" :: "r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}

#define PT_R8(v, i)  "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3]), "=r"(v[i + 4]), "=r"(v[i + 5]), "=r"(v[i + 6]), "=r"(v[i + 7])
#define PT_RW8(v, i) "+r"(v[i]), "+r"(v[i + 1]), "+r"(v[i + 2]), "+r"(v[i + 3]), "+r"(v[i + 4]), "+r"(v[i + 5]), "+r"(v[i + 6]), "+r"(v[i + 7])
#define PT_I8(v, i)  "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3]), "r"(v[i + 4]), "r"(v[i + 5]), "r"(v[i + 6]), "r"(v[i + 7])
__device__ __forceinline__ void pt_ld32(uint32_t * v, uint32_t a) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : PT_R8(v, 0), PT_R8(v, 8), PT_R8(v, 16), PT_R8(v, 24) : "r"(a) : "memory");
}
// the registers of a load are valid only behind the wait: they pass through it, so that no use can be scheduled ahead of it
__device__ __forceinline__ void pt_wait32(uint32_t * v) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : PT_RW8(v, 0), PT_RW8(v, 8), PT_RW8(v, 16), PT_RW8(v, 24) :: "memory");
}
__device__ __forceinline__ void pt_ld16(uint32_t * v, uint32_t a) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];" : PT_R8(v, 0), PT_R8(v, 8) : "r"(a) : "memory");
}
__device__ __forceinline__ void pt_wait16(uint32_t * v) { asm volatile("tcgen05.wait::ld.sync.aligned;" : PT_RW8(v, 0), PT_RW8(v, 8) :: "memory"); }
__device__ __forceinline__ void pt_st16(uint32_t a, const uint32_t * v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" :: "r"(a), PT_I8(v, 0), PT_I8(v, 8) : "memory");
}
__device__ __forceinline__ void pt_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <typename T> __device__ __forceinline__ uint32_t pt_two(float a, float b);
template <> __device__ __forceinline__ uint32_t pt_two<__half>(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *(const uint32_t *) &h; }
template <> __device__ __forceinline__ uint32_t pt_two<__nv_bfloat16>(float a, float b) { const __nv_bfloat162 h = __floats2bfloat162_rn(a, b); return *(const uint32_t *) &h; }
// mask of the halves of w that are infinite or NaN
template <typename T> __device__ __forceinline__ uint32_t pt_odd(uint32_t w) {
    constexpr uint32_t e = sizeof(T) == 2 && std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    return ((w & e) == e ? 0xffffu : 0u) | ((w >> 16 & e) == e ? 0xffff0000u : 0u);
}

// K and V as (dimension, head, token of the page, page) for TMA: boxes of 64 dimensions, one head, `box` tokens.  box = 0: pages that
// a block of BN keys is no multiple or part of (or that no map could be made for): cp.async instead.
struct PtMaps { CUtensorMap k, v; int box; };
__device__ __forceinline__ void pt_tma(uint32_t dst, const CUtensorMap * map, int x, int head, int tok, int page, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
                 :: "r"(dst), "l"(map), "r"(bar), "r"(x), "r"(head), "r"(tok), "r"(page) : "memory");
}
__device__ __forceinline__ void pt_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(bar), "r"(bytes) : "memory");
}

typedef unsigned long long pt_f2;                         // two floats for the packed instructions
__device__ __forceinline__ pt_f2 pt_pair(float a, float b) { pt_f2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ void pt_split(pt_f2 v, float & a, float & b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ pt_f2 pt_mul2(pt_f2 a, pt_f2 b) { pt_f2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ pt_f2 pt_fma2(pt_f2 a, pt_f2 b, pt_f2 c) { pt_f2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ pt_f2 pt_add2(pt_f2 a, pt_f2 b) { pt_f2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
// any + 0 * every value of x
template <typename T> __device__ __forceinline__ float pt_zero_times(uint4 x, float any) {
    const uint32_t w[4] = { x.x, x.y, x.z, x.w };
    uint32_t z = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, __half>::value) { const __half2 y = __hfma2(*(const __half2 *) &w[i], __half2half2(__ushort_as_half(0)), *(const __half2 *) &z); z = *(const uint32_t *) &y; }
        else { const __nv_bfloat162 y = __hfma2(*(const __nv_bfloat162 *) &w[i], __bfloat162bfloat162(__ushort_as_bfloat16(0)), *(const __nv_bfloat162 *) &z); z = *(const uint32_t *) &y; }
    }
    return any + __uint_as_float(pt_odd<T>(z) ? 0x7fffffffu : 0u);
}

// x * 0: NaN stays of what is infinite or NaN
template <typename T> __device__ __forceinline__ void pt_zero(uint4 & x) {
    uint32_t * w = &x.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, __half>::value) { const __half2 y = __hmul2(*(const __half2 *) &w[i], __half2half2(__ushort_as_half(0))); w[i] = *(const uint32_t *) &y; }
        else { const __nv_bfloat162 y = __hmul2(*(const __nv_bfloat162 *) &w[i], __bfloat162bfloat162(__ushort_as_bfloat16(0))); w[i] = *(const uint32_t *) &y; }
    }
}

template <typename T, int D, int BN, int NS, int NTILE, int MIN_CTAS>
__global__ void __launch_bounds__(PT_THREADS(NTILE), MIN_CTAS)
k_paged_attn_tc(const __grid_constant__ PaArgs a, const __grid_constant__ PtMaps maps) {
    using L = PtSmem<D, BN, NS, NTILE>;
    constexpr int COLS = NTILE * (BN + D) <= 128 ? 128 : NTILE * (BN + D) <= 256 ? 256 : 512, NC = D / 8, ROWS = 128 * NTILE, W_MMA = 4 * NTILE;
    extern __shared__ __align__(16) char smem_raw[];
    if (!a.early) chain_wait();                           // behind the store of the same call: only what reads its pages waits (below). No early
                                                          // release: this kernel wants whole SMs
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);      // the shuffle tells the compiler that the warp agrees
    const int failed = pa_failed(a);
    const PaItem item = pa_item(a, blockIdx.x);
    const int seq = item.seq, split = max(item.split, 0), kvh = item.kvh, row0 = item.tile * ROWS, chunk = item.split < 0 ? 1 << 30 : a.chunk;
    const PaSeq s = pa_seq(a, seq);
    const int n_rows = s.n_new * a.group;
    const int k0 = split * chunk, k1 = row0 < n_rows ? min(pa_reach(a, s, row0), k0 + chunk) : 0;
    if (row0 >= n_rows || failed || (k0 >= k1 && split != 0)) {      // no rows, or an empty split, which the join does not read
        // What follows waits for this launch only, which therefore must not end before the store, not even where no sequence has a new token.  One
        // CTA sees to that: with all of those that have no rows, ragged prompts took 35.3 us instead of 34.4.
        if (a.early && blockIdx.x == 0) chain_wait();
        return;
    }
    // blocks of each tile; a tile without rows has none
    int n_blk[NTILE], sure[NTILE];                               // sure: keys below are seen by every row of the tile
#pragma unroll
    for (int t = 0; t < NTILE; ++t) {
        const int r0 = row0 + t * 128, r1 = min(r0 + 128, n_rows);
        const int reach = r0 >= n_rows ? 0 : a.causal ? min(s.len, max(s.len - s.n_new + (r1 - 1) / a.group + 1, 0)) : s.len;
        n_blk[t] = (max(min(reach, k0 + chunk) - k0, 0) + BN - 1) / BN;
        sure[t] = a.causal ? s.len - s.n_new + r0 / a.group + 1 : s.len;
    }
    const int n = NTILE == 1 ? n_blk[0] : max(n_blk[0], n_blk[NTILE - 1]);
    char * smem = smem_raw + ((1024 - ((uint32_t) __cvta_generic_to_shared(smem_raw) & 1023)) & 1023);
    const uint32_t sb = (uint32_t) __cvta_generic_to_shared(smem);
    const uint32_t k_full = sb + L::BAR, k_empty = k_full + 8 * NS, v_full = k_empty + 8 * NS, v_empty = v_full + 8 * NS, v_here = v_empty + 8 * NS,
                   q_full = v_here + 8 * NS, s_full = q_full + 8, p_full = s_full + 16, o_full = p_full + 16;
    uint32_t * tmem_slot = (uint32_t *) (smem + L::MISC);
    volatile int * abort_flag = (volatile int *) (smem + L::MISC + 4);
    volatile int * odd_flag = (volatile int *) (smem + L::MISC + 8);
    if (tid == 0) {
        auto init = [](uint32_t bar, int count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(bar), "r"(count)); };
        for (int i = 0; i < 5 * NS; ++i) init(k_full + 8 * i, 1);
        init(q_full, 4 * NTILE);
        for (int t = 0; t < NTILE; ++t) { init(s_full + 8 * t, 1); init(p_full + 8 * t, 4); init(o_full + 8 * t, 1); }
        *abort_flag = 0;
        *odd_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == W_MMA) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(sb + L::MISC), "n"(COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pt_before();
    __syncthreads();
    pt_after();
    const uint32_t tmem = *tmem_slot;

    if (warp < W_MMA) {
        // ================= softmax =================
        const int t = NTILE == 1 ? 0 : warp >> 2, r = (warp & 3) * 32 + lane, row = row0 + t * 128 + r;
        const bool valid = row < n_rows;
        const int tok = valid ? row / a.group : 0, head = kvh * a.group + (valid ? row % a.group : 0);
        {
            const uint32_t flip = a.scale_log2 < 0 ? 0x80008000u : 0;   // a negative scale goes into the signs of Q: the maximum is then one of S
            const char * q = a.q + (s.tok0 + tok) * a.nb_q_tok + head * a.nb_q_head;
            char * dst = smem + L::Q + t * L::QT + r * 128;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                uint4 x = make_uint4(0, 0, 0, 0);
                if (valid) { x = *(const uint4 *) (q + c * 16); x.x ^= flip; x.y ^= flip; x.z ^= flip; x.w ^= flip; if (a.scale_log2 == 0) pt_zero<T>(x); }
                *(uint4 *) (dst + (c >> 3) * 128 * 128 + (((c & 7) ^ (r & 7)) << 4)) = x;
            }
            pt_proxy_fence();
            __syncwarp();
            if (lane == 0) pt_arrive(q_full);
        }
        if (a.early) chain_wait();
        const float scale = a.scale_log2 == 0 ? 1.0f : fabsf(a.scale_log2);        // 0 is in Q: masked scores are -inf, and -inf * 0 is not
        const int last = !valid ? -1 : a.causal ? s.len - s.n_new + tok : s.len - 1;
        const uint32_t lanes = (uint32_t) (warp & 3) << 21;              // 32 lanes per warp, in bits 16 and up
        const uint32_t ts = tmem + lanes + t * BN, to = tmem + lanes + NTILE * BN + t * D;
        float m = -INFINITY, l = 0.0f;
        for (int j = 0; j < n_blk[t]; ++j) {
            if (!pt_wait_warp(s_full + 8 * t, j & 1, abort_flag, 1)) goto done;
            pt_after();
            const int seen = last + 1 - (k0 + j * BN);                   // this row sees the block's first `seen` keys
            const bool edge = k0 + (j + 1) * BN > sure[t];
            // Two copies for head_dim 128, so that blocks which every row sees wholly hold no code for masks (chunk of 2048 over 16k keys, with the weights of
            // the time: 955 -> 932 us); one for head_dim 64, whose four CTAs an SM share the instruction cache (ragged prompts: 36.1 against 37.4 us with two).
            auto block = [&](auto masked) {
                // 32 scores at a time, read once for the maximum and once for the weights: keeping 64, 96 or 128 of them in registers between
                // the two was no faster
                auto scores = [&](uint32_t * y, int c) {
                    pt_ld32(y, ts + c);
                    pt_wait32(y);
                    if (decltype(masked)::value && (NTILE > 1 || edge)) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) if (c + i >= seen) y[i] = 0xff800000u;
                    }
                };
                float m4[4] = { -INFINITY, -INFINITY, -INFINITY, -INFINITY };
#pragma unroll
                for (int c = 0; c < BN; c += 32) {
                    uint32_t y[32];
                    scores(y, c);
#pragma unroll
                    for (int i = 0; i < 32; i += 8)
#pragma unroll
                        for (int u = 0; u < 4; ++u) m4[u] = fmaxf(m4[u], fmaxf(__uint_as_float(y[i + u]), __uint_as_float(y[i + 4 + u])));
                }
                const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
                const bool grow = (mx - m) * scale > PtLag<T>::lag;                // also when there was no key so far; -inf - -inf is not
                if (__any_sync(0xffffffffu, grow)) {
                    const float m1 = fmaxf(m, mx), f = m1 == -INFINITY ? 1.0f : pa_exp2((m - m1) * scale);
                    m = m1;
                    l *= f;
                    if (j > 0) {
#pragma unroll 1
                        for (int c = 0; c < D; c += 16) {
                            uint32_t o[16];
                            pt_ld16(o, to + c);
                            pt_wait16(o);
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                            pt_st16(to + c, o);
                        }
                    }
                }
                // difference first: exact where it matters, whatever the scores' size.  s * scale - m in one operation is 1.6% faster, but off by
                // the rounding of m, which is a large number where the scores are (1e36: infinite weights)
                const float base = m == -INFINITY ? 0.0f : -m;
                const pt_f2 scale2 = pt_pair(scale, scale), base2 = pt_pair(base, base), raise2 = pt_pair(PtLag<T>::raise, PtLag<T>::raise);
                pt_f2 l2[2] = { 0ull, 0ull };
#pragma unroll
                for (int c = 0; c < BN; c += 32) {
                    uint32_t w[16], y[32];
                    scores(y, c);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float y0, y1;
                        const pt_f2 d = pt_add2(pt_pair(__uint_as_float(y[2 * i]), __uint_as_float(y[2 * i + 1])), base2);
                        pt_split(PtLag<T>::raise == 0.0f ? pt_mul2(d, scale2) : pt_fma2(d, scale2, raise2), y0, y1);
                        y0 = pa_exp2(y0); y1 = pa_exp2(y1);
                        l2[i & 1] = pt_add2(l2[i & 1], pt_pair(y0, y1));
                        w[i] = pt_two<T>(y0, y1);
                    }
                    pt_st16(ts + c / 2, w);
                }
                float l0, l1;
                pt_split(pt_add2(l2[0], l2[1]), l0, l1);
                l += l0 + l1;
            };
            if (edge || NTILE == 1) block(std::true_type());
            else block(std::false_type());
            pt_wait_st();
            pt_before();
            __syncwarp();
            if (lane == 0) pt_arrive(p_full + 8 * t);
        }
        if (n_blk[t] > 0) {
            if (!pt_wait_warp(o_full + 8 * t, 0, abort_flag, 2)) goto done;
            pt_after();
        }
        m *= scale;                                                       // of the scores so far; from here on an exponent of two
        const int64_t out = (s.tok0 + tok) * a.n_head + head;
        const bool odd = n_blk[t] > 0 && *odd_flag;
        const bool whole = item.split < 0;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        l *= PtLag<T>::lower;
        char * dst = a.dst + (s.tok0 + tok) * a.nb_dst_tok + head * a.nb_dst_head;
        float * part = a.part + (item.slot * ROWS + t * 128 + r) * (D + 4);
#pragma unroll 1
        for (int c = 0; c < D; c += 16) {
            uint32_t o[16];
            if (n_blk[t] > 0) { pt_ld16(o, to + c); pt_wait16(o); }
            else {
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] = 0;
            }
            if (odd && valid) {                                           // values that were taken out of V tiles, for the rows that see them
                for (int key = k0 + max(0, sure[0] - k0) / BN * BN; key <= min(last, k0 + n_blk[t] * BN - 1); ++key) {
                    const int page = a.tables[seq * a.table_stride + key / a.page_size];
                    if (page < 0 || page >= a.n_pages) continue;
                    const T * v = (const T *) (a.v + page * a.nb_page + (key % a.page_size) * a.nb_tok + kvh * a.nb_head) + c;
#pragma unroll
                    for (int i = 0; i < 16; ++i) { const float y = (float) v[i]; if (!(fabsf(y) < INFINITY)) o[i] = __float_as_uint(__uint_as_float(o[i]) + y); }
                }
            }
            if (!valid) continue;
            if (!whole) {
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    float4 x = make_float4(__uint_as_float(o[i]), __uint_as_float(o[i + 1]), __uint_as_float(o[i + 2]), __uint_as_float(o[i + 3]));
                    x.x *= PtLag<T>::lower; x.y *= PtLag<T>::lower; x.z *= PtLag<T>::lower; x.w *= PtLag<T>::lower;
                    *(float4 *) (part + c + i) = x;
                }
            } else {
                uint32_t w[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = pt_two<T>(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
                *(uint4 *) (dst + c * 2) = make_uint4(w[0], w[1], w[2], w[3]);
                *(uint4 *) (dst + c * 2 + 16) = make_uint4(w[4], w[5], w[6], w[7]);
            }
        }
        if (valid && !whole) { part[D] = m; part[D + 1] = l; }
        if (valid && whole && a.lse) a.lse[out] = l == 0.0f ? -INFINITY : m * 0.69314718f + logf(l);
    } else if (warp == W_MMA) {
        // ================= MMA issue =================
        if (lane == 0 && n > 0) {
            constexpr uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1u << 7 | 1u << 10 : 0u;
            constexpr uint32_t id_s = 1u << 4 | type | (uint32_t) (BN >> 3) << 17 | 128u >> 4 << 24;
            constexpr uint32_t id_o = 1u << 4 | type | 1u << 16 | (uint32_t) (D >> 3) << 17 | 128u >> 4 << 24;
            auto scores = [&](int t, int j) {
                const uint32_t q = sb + L::Q + t * L::QT, k = sb + L::K + (j % NS) * L::TILE;
#pragma unroll
                for (int i = 0; i < D / 16; ++i)
                    pt_mma_ss(tmem + t * BN, pt_desc(q + (i >> 2) * 128 * 128 + (i & 3) * 32, 16), pt_desc(k + (i >> 2) * BN * 128 + (i & 3) * 32, 16), id_s, i > 0);
                pt_commit(s_full + 8 * t);
            };
            if (!pt_wait(q_full, 0, abort_flag, 3) || !pt_wait(k_full, 0, abort_flag, 4)) goto done;
            pt_after();
            for (int t = 0; t < NTILE; ++t) if (n_blk[t] > 0) scores(t, 0);
            pt_commit(k_empty);
            for (int j = 0; j < n; ++j) {
                if (!pt_wait(v_full + 8 * (j % NS), j / NS & 1, abort_flag, 5)) goto done;
                if (j + 1 < n && !pt_wait(k_full + 8 * ((j + 1) % NS), (j + 1) / NS & 1, abort_flag, 6)) goto done;
                for (int t = 0; t < NTILE; ++t) {
                    if (j >= n_blk[t]) continue;
                    if (!pt_wait(p_full + 8 * t, j & 1, abort_flag, 7)) goto done;
                    pt_after();
                    const uint32_t v = sb + L::V + (j % NS) * L::TILE;
#pragma unroll
                    for (int i = 0; i < BN / 16; ++i) pt_mma_ts(tmem + NTILE * BN + t * D, tmem + t * BN + i * 8, pt_desc(v + i * 2048, BN * 128), id_o, j > 0 || i > 0);
                    if (j + 1 < n_blk[t]) scores(t, j + 1);
                    else pt_commit(o_full + 8 * t);
                }
                pt_commit(v_empty + 8 * (j % NS));
                if (j + 1 < n) pt_commit(k_empty + 8 * ((j + 1) % NS));
            }
        }
    } else {
        // ================= K and V =================
        if (a.early) chain_wait();
        const bool is_v = warp == W_MMA + 2;
        const char * base = (is_v ? a.v : a.k) + kvh * a.nb_head;
        const uint32_t ring = sb + (is_v ? L::V : L::K), full = is_v ? v_full : k_full, empty = is_v ? v_empty : k_empty;
        const int32_t * table = a.tables + seq * a.table_stride;
        constexpr int G = BN / 32;
        const int box = maps.box;
        // V's non-finite values, in blocks that are not wholly seen, are taken out; a lane looks at the same 16-byte chunks that it copies
        auto clean = [&](int jj) {
            auto place = [&](int g, int c) {
                const int i = c * 32 + lane, r = i / NC, ch = i % NC;
                return (uint4 *) (smem + L::V + (jj % NS) * L::TILE + (ch >> 3) * BN * 128 + (g * 32 + r) * 128 + (((ch & 7) ^ (r & 7)) << 4));
            };
            float any = 0.0f;                                             // NaN as soon as a value is infinite or NaN: x * 0
            const int rows = k1 - (k0 + jj * BN);                         // behind them nobody looks: zeros, whatever the page holds
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    if (g * 32 + (c * 32 + lane) / NC < rows) any = pt_zero_times<T>(*place(g, c), any);
                    else *place(g, c) = make_uint4(0, 0, 0, 0);
                }
            if (any != any) {
#pragma unroll 1
                for (int g = 0; g < G; ++g)
#pragma unroll 1
                    for (int c = 0; c < NC; ++c) {
                        uint4 * p = place(g, c);
                        uint4 x = *p;
                        x.x &= ~pt_odd<T>(x.x); x.y &= ~pt_odd<T>(x.y); x.z &= ~pt_odd<T>(x.z); x.w &= ~pt_odd<T>(x.w);
                        *p = x;
                    }
                *odd_flag = 1;
            }
            pt_proxy_fence();
        };
        if (box) {
            // TMA: lane i brings the block's i-th page (or its part of one); pages out of reach or out of the pool are named n_pages, which
            // reads as zeros.  A page's tokens behind the sequence's end come along: K's are masked, V's cleaned.
            const int per = BN / box;
            auto page_of = [&](int j) {
                const int key = k0 + j * BN + lane * box;
                if (j >= n || lane >= per || key >= k1) return a.n_pages;
                const int p = table[key / a.page_size];
                return p < 0 || p > a.n_pages ? a.n_pages : p;
            };
            int page = page_of(0);
            for (int j = 0; j < n; ++j) {
                const int now = page;
                page = page_of(j + 1);
                if (!pt_wait_warp(empty + 8 * (j % NS), (j / NS & 1) ^ 1, abort_flag, 8)) {
                    for (int i = max(0, j - NS); i < j; ++i) pt_poll((is_v ? v_here : k_full) + 8 * (i % NS), i / NS & 1);       // copies under way
                    goto done;
                }
                const uint32_t bar = (is_v ? v_here : k_full) + 8 * (j % NS), dst = ring + (j % NS) * L::TILE + lane * box * 128;
                if (lane == 0) pt_expect(bar, L::TILE);
                __syncwarp();
                if (lane < per) {
                    const int tok = (k0 + j * BN + lane * box) % a.page_size;
#pragma unroll
                    for (int h = 0; h < D / 64; ++h) pt_tma(dst + h * BN * 128, is_v ? &maps.v : &maps.k, h * 64, kvh, tok, now, bar);
                }
                __syncwarp();
                if (is_v) {
                    if (!pt_wait_warp(bar, j / NS & 1, abort_flag, 9)) goto done;
                    if (k0 + (j + 1) * BN > sure[0]) clean(j);
                    __syncwarp();
                    if (lane == 0) pt_arrive(v_full + 8 * (j % NS));
                }
            }
            if (!is_v)                                                    // nothing may be under way when the CTA ends
                for (int j = max(0, n - NS); j < n; ++j) if (!pt_wait_warp(k_full + 8 * (j % NS), j / NS & 1, abort_flag, 10)) break;
            goto done;
        }
        int page[G];
        auto look = [&](int j) {
#pragma unroll
            for (int g = 0; g < G; ++g) { const int key = k0 + j * BN + g * 32 + lane; page[g] = j < n && key < k1 ? table[key / a.page_size] : -1; }
        };
        look(0);
        for (int j = 0; j < n; ++j) {
            const uint32_t dst = ring + (j % NS) * L::TILE;
            int64_t at[G];
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const int key = k0 + j * BN + g * 32 + lane;
                at[g] = page[g] >= 0 && page[g] < a.n_pages ? page[g] * a.nb_page + (key % a.page_size) * a.nb_tok : -1;
                asm volatile("" : "+l"(at[g]));       // kept: computed again for every chunk otherwise, division included (30 000 cycles a block)
            }
            look(j + 1);
            if (!pt_wait_warp(empty + 8 * (j % NS), (j / NS & 1) ^ 1, abort_flag, 8)) goto done;
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const int i = c * 32 + lane, r = i / NC, ch = i % NC;        // row of the group, 16-byte chunk of the row
                    const int64_t off = __shfl_sync(0xffffffffu, at[g], r);
                    const uint32_t d = dst + (ch >> 3) * BN * 128 + (g * 32 + r) * 128 + (((ch & 7) ^ (r & 7)) << 4);
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(d), "l"(base + (off < 0 ? 0 : off + ch * 16)), "r"(off < 0 ? 0 : 16) : "memory");
                }
            asm volatile("cp.async.commit_group;" ::: "memory");
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            if (is_v && k0 + (j + 1) * BN > sure[0]) clean(j);
            pt_proxy_fence();
            __syncwarp();
            if (lane == 0) pt_arrive(full + 8 * (j % NS));
        }
    }
done:
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
    pt_before();
    __syncthreads();
    if (warp == W_MMA) {
        pt_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "n"(COLS) : "memory");
    }
}

typedef CUresult (*pt_encode_fn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *, const cuuint32_t *,
                                 CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static pt_encode_fn pt_encode() {
    static const pt_encode_fn f = [] {
        void * p = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &r) != cudaSuccess || r != cudaDriverEntryPointSuccess) { cudaGetLastError(); p = nullptr; }
        return (pt_encode_fn) p;
    }();
    return f;
}

// maps.box = 0 where the page size does not fit TMA boxes of whole 8-row groups, or the driver makes no map
static void pt_make_maps(PtMaps & m, const PaArgs & a, int D, int BN, bool f16) {
    memset(&m, 0, sizeof(m));
    const int ps = a.page_size, box = ps < BN ? ps : BN;
    if (ps % 8 || (ps < BN ? BN % ps : ps % BN) || !pt_encode()) return;
    const cuuint64_t dims[4] = { (cuuint64_t) D, (cuuint64_t) a.n_head_kv, (cuuint64_t) ps, (cuuint64_t) a.n_pages };
    const cuuint64_t row = (cuuint64_t) D * 2;
    const cuuint64_t strides[3] = { a.n_head_kv > 1 ? (cuuint64_t) a.nb_head : row, (cuuint64_t) a.nb_tok, (cuuint64_t) a.nb_page };
    const cuuint32_t size[4] = { 64, 1, (cuuint32_t) box, 1 }, one[4] = { 1, 1, 1, 1 };
    for (int i = 0; i < 2; ++i)
        if (pt_encode()(i ? &m.v : &m.k, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, (void *) (i ? a.v : a.k), dims, strides, size, one,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) return;
    m.box = box;
}

template <typename T, int D, int BN, int NS, int NTILE, int MIN_CTAS>
static cudaError_t pt_go(const PaArgs & a, int64_t n_items, cudaStream_t st) {
    static_assert(128 * NTILE == PA_TC_ROWS(D) && BN == PA_TC_KEYS(D) && MIN_CTAS == PA_TC_CTAS(D), "what the plan counts with");
    constexpr auto k = k_paged_attn_tc<T, D, BN, NS, NTILE, MIN_CTAS>;
    constexpr int smem = PtSmem<D, BN, NS, NTILE>::BYTES;
    cudaError_t e = allow_once<k>(smem);
    if (e != cudaSuccess) return e;
    PtMaps maps;
    pt_make_maps(maps, a, D, BN, std::is_same<T, __half>::value);
    const int64_t ctas = a.n_whole + (n_items - a.n_whole) * a.n_split;
    e = launch_chained(k, dim3((unsigned) ctas), dim3(PT_THREADS(NTILE)), smem, st, a, maps);
    if (e == cudaSuccess) B200_LAUNCHED();
    return e;
}

cudaError_t pa_tc_launch(const PaArgs & a, int head_dim, int type, int64_t n_items, cudaStream_t st) {
    if (head_dim == 64) return type == B200_TYPE_F16 ? pt_go<__half, 64, 64, 2, 1, 4>(a, n_items, st) : pt_go<__nv_bfloat16, 64, 64, 2, 1, 4>(a, n_items, st);
    return type == B200_TYPE_F16 ? pt_go<__half, 128, 128, 2, 2, 1>(a, n_items, st) : pt_go<__nv_bfloat16, 128, 128, 2, 2, 1>(a, n_items, st);
}
