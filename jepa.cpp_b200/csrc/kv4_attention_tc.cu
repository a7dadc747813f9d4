// Attention over the paged 4-bit cache for many rows (kv4.h; the formula is in kv4_attention.cu): tcgen05 products.
//
// One CTA per (request, cache head, 256 columns, range of keys); a column is a (new token, head of the group) pair, a
// row of the two 128-row tiles here. Keys come in blocks of 64. Warps:
//   0 .. 7   softmax: one thread per row (4 warps a tile, one per TMEM lane quadrant). They put the queries in place
//            once (scaled by a power of two into f16's range), then per block read their row of S = Q K^T from
//            TMEM once, and put the weights P = 2^(s - z) back in f16 over the front half of S's
//            columns, where the second product takes it as its A operand: P never passes through shared memory.
//            O stays in TMEM; it is rescaled only when a weight would pass 2^14.5 (they start from 2^6 .. 2^7 at the
//            largest, and f16 ends at 2^16).
//   8 .. 11  conversion from 4 bits to d (c - 8) in f16 (exact, kv4.h), one thread per row: two warps for K, two for V,
//            written in the 128-byte swizzle of the products' operands (K: K-major; V: MN-major, keys down
//            the rows). The next block's codes are loaded before this one's are converted; four blocks are held.
//   12, 13   issue the products of tile 0 and 1: S_t = Q_t K^T (M 128, N 64), two blocks ahead in two buffers, and
//            O_t += P_t V (M 128, N hd). Softmax never waits for a product of its own block, and the tiles run on
//            their own.
// Up to head_dim 64 TMEM holds Q beside S and O, above that Q stays in shared memory. The tensor core reads shared memory, and A
// in TMEM, at about 64 bytes a cycle each: a 128 x 64 x 16 product takes 64 cycles with Q in TMEM and 100 with Q in shared
// memory, 128 x 128 x 16 (P V at head_dim 128) 64. What bounds it: at head_dim 128 the products, 2100 of the 2700 cycles a pair
// of tiles takes for 64 keys (chunks of 700 .. 2047 rows behind 4100 .. 8191 keys, 32 / 8 heads: 698 us, 704 TFLOP/s); at
// head_dim 64 the softmax, 1024 of 2300 cycles of which are exponentials, and what a CTA takes whatever its keys (queries,
// tensor memory, first codes, stores): 96 x 256 rows of 16 heads take 91 us and 12 us for every 64 keys, 247 us for 774, which
// is 17,000 cycles a CTA and 2250 for every 64 keys (258 rows: 287 us, the rows kernel takes the last 2).
// Registers: 118 to 128, with 48 bytes of spills at head_dim 128 and 8 at 96.
// Measured and not taken, at head_dim 128: 128 keys a block with one buffer of S, 784 us or more (the softmax waits 2200 cycles
// a block); Q in TMEM with one buffer, 858; two blocks' scores in one product of N 128, 884; turns of the two tiles' exponentials,
// 756 against 742; a quarter of the exponentials as polynomials, no change (head_dim 64: 301 instead of 312).
// Within 8 channels the operands keep the order in which codes unpack, 0 4 1 5 2 6 3 7: Q is written in the order of
// K's words, O's columns are put right when they are stored.
// TMEM columns: O_0, O_1 (hd each), Q_0, Q_1 (hd / 2) up to head_dim 64, then two buffers of S a tile.
// A value scale that is not finite enters as zeros; the rows that see such a key get NaN in that group at the end, so a NaN
// behind a row's mask does not reach it (0 * NaN).
// Every mbarrier wait is bounded: when one runs out the CTA raises the error flag, waits for the products that it has issued,
// writes NaN to the rows that it has not finished, and ends.
#include "kv4_device.h"
#include "common.h"
#include "launch.h"
#include "tcgen05.cuh"

#include <atomic>
#include <cfloat>

namespace jb {

// The wait that ran out last, and how many CTAs have given up one. The device only counts; the host remembers how far it has told
// (kv4_error_flag), so that what is raised while another thread or stream reads is told the next time.
struct Kv4Failures { int code; unsigned count; };
__device__ Kv4Failures g_kv4_failures = {0, 0};

namespace {

using namespace tc;

constexpr int BLK = 64;                         // keys per block
constexpr int STAGES = 4;                       // blocks of K and of V in shared memory
constexpr int SOFT = 8, CONV = 4, PROD = 2;     // warps of each kind
constexpr int THREADS = 32 * (SOFT + CONV + PROD);
constexpr uint32_t QATOM = 128 * 128, ATOM = BLK * 128;     // bytes of 128 and of BLK rows of 64 f16
constexpr int SLOTS = 8;                        // blocks whose key masks are kept: those in shared memory, and two that
                                                // have left it as operands but not yet as scores (S of block j - STAGES is
                                                // done: the weights of block j - STAGES - 2 are there, its masks are read)

__host__ __device__ constexpr uint32_t idesc(int n, bool b_mn_major) {      // kind::f16, f16 in, f32 out, M 128
    return (1u << 4) | ((uint32_t) (n >> 3) << 17) | ((uint32_t) (128 >> 4) << 24) | (b_mn_major ? 1u << 16 : 0u);
}
// MN-major operand in the 128-byte swizzle: 64-element columns of atoms one block of rows (ATOM bytes) apart (LBO),
// 8-row groups 1024 bytes apart (SBO)
__device__ __forceinline__ uint64_t mn_desc(uint32_t saddr) {
    uint64_t d = sw128_desc(saddr) & ~((uint64_t) 0x3FFF << 16);
    return d | (uint64_t) (ATOM >> 4) << 16;
}
// The products take a descriptor's words apart: only the low one (address) changes within a block, by constants.
// D (+)= A B, A in shared memory / in tensor memory
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "setp.ne.b32 p, %6, 0;\n\tmov.b64 da, {%1, %2};\n\tmov.b64 db, {%3, %4};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n\t}"
        :: "r"(d), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(id), "r"(acc));
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t b_hi, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
        "setp.ne.b32 p, %5, 0;\n\tmov.b64 db, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}"
        :: "r"(d), "r"(a), "r"(b_lo), "r"(b_hi), "r"(id), "r"(acc));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        :: "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
           "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// all threads of the CTA, from any branch
__device__ __forceinline__ void cta_sync() {
    fence_before();
    asm volatile("barrier.sync 0;" ::: "memory");
    fence_after();
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void st_shared16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" :: "r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// one lane of a converged warp (products issued under lane == 0 instead took 120 cycles each to issue)
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}

struct Args : Kv4Attn { Kv4Waits waits; };

// the whole warp waits, and agrees on the outcome
__device__ __forceinline__ bool warp_wait(const Args & a, uint64_t * bar, uint32_t parity, int code) {
    if (code == a.waits.give_up_at) {
        atomicExch(&g_kv4_failures.code, code);
        return false;
    }
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, code, &g_kv4_failures.code, a.waits.limit));
}

// bits of an f16 infinity or NaN
__device__ __forceinline__ bool not_finite(uint32_t h) { return (h & 0x7c00u) == 0x7c00u; }
// the low n bits
__device__ __forceinline__ uint32_t seen(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }

template <int NG> __host__ __device__ constexpr int atoms() { return (NG + 1) / 2; }
template <int NG> constexpr size_t tiles_smem() { return (size_t) atoms<NG>() * ((NG <= 2 ? 0 : 2 * QATOM) + 2 * STAGES * ATOM) + 1024; }

template <class T, int NG>
__global__ void __launch_bounds__(THREADS, 1) k_kv4_tiles(const Kv4Pool pool, const Args a, const Split sp, int tiles, int vec) {
    constexpr int HD = 32 * NG, AT = atoms<NG>(), W = 4 * NG;      // W: 8-channel words of a row
    constexpr bool QT = NG <= 2;                                   // Q in tensor memory, else in shared memory
    constexpr int NB = 2;                                          // buffers of S a tile
    constexpr uint32_t Q_COL = 2 * HD, S_COL = QT ? 3 * HD : 2 * HD;
    static_assert(S_COL + 2 * NB * BLK <= 512, "tensor memory");
    extern __shared__ uint8_t smem_raw[];
    // shared addresses
    const uint32_t sQ = (smem_u32(smem_raw) + 1023) & ~1023u, sK = sQ + (QT ? 0 : 2 * AT * QATOM), sV = sK + STAGES * AT * ATOM;
    struct Bars {
        uint64_t k_full[STAGES], v_full[STAGES], k_empty[2][STAGES], v_empty[2][STAGES], s_full[2][NB], p_full[2][NB], o_done[2][NB];   // [tile][stage or buffer]
        uint64_t drained[2];
    };
    __shared__ __align__(8) Bars bars;
    // per block and 32 keys: any exception; keys without a page; keys whose value scale of a group is not finite
    __shared__ __align__(16) uint32_t s_any[SLOTS][2], s_hole[SLOTS][2], s_bad[SLOTS][NG][2];
    __shared__ uint32_t tmem_sh;
    __shared__ int abort_sh;
    asm volatile("griddepcontrol.wait;" ::: "memory");

    const int warp = __shfl_sync(0xffffffffu, (int) (threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int kh = blockIdx.y / tiles, r = blockIdx.z, G = a.heads / pool.heads;
    const Req rq = request_of(a, pool.page_shift, r);
    const int n_cols = tile_columns((rq.row1 - rq.row0) * G);
    const int span = sp.span(rq.len), used = sp.used(rq.len);
    if (n_cols <= 0 || (int) (blockIdx.y % tiles) * 256 >= n_cols || (blockIdx.x && (int) blockIdx.x >= used)) return;
    const int k0 = blockIdx.x * span, k1 = range_end(rq.len, k0, span);

    if (warp == SOFT) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(&tmem_sh)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (threadIdx.x == 0) abort_sh = 0;

    int c0 = (int) (blockIdx.y % tiles) * 256;
    for (; c0 < n_cols; c0 += tiles * 256) {
        const int cols = min(256, n_cols - c0), n_tiles = cols > 128 ? 2 : 1;
        const int kend = min(visible(rq, rq.row0 + (c0 + cols - 1) / G, a.frame), k1);   // the last row sees most
        const int nb_all = kend > k0 ? (kend - k0 + BLK - 1) / BLK : 0;
        const int kend0 = n_tiles == 1 ? kend : min(visible(rq, rq.row0 + (c0 + 127) / G, a.frame), kend);
        const int nb0 = kend0 > k0 ? (kend0 - k0 + BLK - 1) / BLK : 0;          // blocks of tile 0
        if (threadIdx.x == THREADS - 1) {
            for (int s = 0; s < STAGES; s++) {
                mbar_init(&bars.k_full[s], CONV / 2);
                mbar_init(&bars.v_full[s], CONV / 2);
                for (int t = 0; t < 2; t++) { mbar_init(&bars.k_empty[t][s], 1); mbar_init(&bars.v_empty[t][s], 1); }
            }
            for (int t = 0; t < 2; t++) {
                mbar_init(&bars.drained[t], 1);
                // (one a buffer: a warp may be as many blocks ahead of another)
                for (int i = 0; i < NB; i++) {
                    mbar_init(&bars.s_full[t][i], 1);
                    mbar_init(&bars.o_done[t][i], 1);
                    mbar_init(&bars.p_full[t][i], (uint32_t) max(1, (min(128, cols - 128 * t) + 31) / 32));
                }
            }
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            fence_async();
        }
        // ---- queries: first as they are into the stages' memory, by consecutive threads along the rows (a thread a row took
        // 32 cache lines a load, 8,000 to 15,000 cycles in all), then thread = row of the tiles
        constexpr int QB = 5;                   // words a thread has on their way at a time
        for (int i0 = threadIdx.x; i0 < 256 * W; i0 += QB * THREADS) {
            uint4 v[QB];
#pragma unroll
            for (int u = 0; u < QB; u++) {
                const int i = i0 + u * THREADS, cc = c0 + i / W;
                v[u] = make_uint4(0, 0, 0, 0);
                if (i < 256 * W && cc < n_cols) {
                    const T * q = (const T *) a.q + (long long) (rq.row0 + cc / G) * a.q_tok + (kh * G + cc % G) * a.q_head + 8 * (i % W);
                    if (vec & 1) {
                        v[u] = *(const uint4 *) q;
                    } else {
                        T e[8];
#pragma unroll
                        for (int k = 0; k < 8; k++) e[k] = q[k];
                        memcpy(&v[u], e, 16);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < QB; u++) {
                const int i = i0 + u * THREADS, rr = i / W, c = i % W;
                if (i < 256 * W) st_shared16(sK + rr * (2 * HD) + ((c ^ (rr & 3)) << 4), v[u].x, v[u].y, v[u].z, v[u].w);
            }
        }
        cta_sync();                             // TMEM is there, and free of the columns before
        // (not earlier: launch.h; a CTA that left above releases them by its end)
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
        const uint32_t tmem = tmem_sh;
        float f = 0.0f;                         // of this row's scores, in log2 units
        int lim = 0;                            // keys this row sees
        const int col = c0 + threadIdx.x;
        const int row = rq.row0 + (warp < SOFT && col < n_cols ? col / G : 0), head = kh * G + (col < n_cols ? col % G : 0);
        if (warp < SOFT) {
            const bool there = col < n_cols;
            const uint32_t mine = sK + threadIdx.x * (2 * HD);
            auto word = [&](int s, float (&x)[8]) {         // words in the order of the key rows
                T e[8];
                const uint4 v = ld_shared16(mine + (((4 * (s % NG) + s / NG) ^ (lane & 3)) << 4));
                memcpy(e, &v, 16);
#pragma unroll
                for (int c = 0; c < 8; c++) x[c] = from_type(e[c]);
            };
            float amax = 0.0f, x[8];
#pragma unroll
            for (int s = 0; s < W; s++) {
                word(s, x);
#pragma unroll
                for (int c = 0; c < 8; c++) amax = fmaxf(amax, fabsf(x[c]));
            }
            int ex = 0;
            const int eb = (int) (__float_as_uint(amax) >> 23);
            if (amax > 0.0f && eb < 255) ex = min(14 - (eb - 127), 126);
            const float up = __int_as_float((127 + ex) << 23) * (a.scale < 0.0f ? -1.0f : 1.0f);    // f >= 0 below
            // (not 0, which would make NaN of a masked score's -inf)
            f = fmaxf(fabsf(a.scale) * 1.4426950408889634f * __int_as_float((127 - ex) << 23), 1e-37f);
            if (there) lim = min(visible(rq, row, a.frame), kend);
            const uint32_t qc = tmem + ((uint32_t) (32 * (warp & 3)) << 16) + Q_COL + (warp >> 2) * (HD / 2);
            const uint32_t qs = sQ + (warp >> 2) * AT * QATOM + (threadIdx.x & 127) * 128;
#pragma unroll
            for (int s = 0; s < W; s += 4) {
                uint32_t w[16];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    word(s + i, x);
#pragma unroll
                    for (int c = 0; c < 4; c++) w[4 * i + c] = pack_h2(x[c] * up, x[c + 4] * up);
                    if (!QT) st_shared16(qs + ((s + i) / 8) * QATOM + ((((s + i) & 7) ^ (lane & 7)) << 4), w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                }
                if (QT) tmem_st16(qc + 4 * s, w);
            }
            tmem_wait_st();
            fence_async();                      // queries in shared memory
        }

        if (warp >= SOFT && warp < SOFT + CONV) {
            // ---- conversion: thread = a K row (warps 8, 9) or a V row (10, 11) of the block
            const int kt = threadIdx.x & (BLK - 1), cw = warp & 1;
            const bool keys = warp < SOFT + 2;
            const int32_t * table = a.table + (size_t) r * a.width;
            const int n_pages = (int) (pool.n_slots >> pool.page_shift), pmask = (1 << pool.page_shift) - 1, P = 1 << pool.page_shift;
            // this head's rows and scales of page 0, and from page to page
            const uint32_t d_plane = ((uint32_t) pool.heads * NG) << pool.page_shift, q_page = ((uint32_t) pool.heads << pool.page_shift) * 32 * NG;
            const uint8_t * q_head = pool.q + kv4_q_at(pool, 0, keys ? 0 : 1, kh, 0);
            const uint16_t * d_head = (const uint16_t *) pool.d + kv4_d_at(pool, 0, keys ? 0 : 1, kh, 0);
            // (a table entry is loaded a block before it is used and checked; volatile keeps the load there. With this, the scales
            // in 32 bits each and no choice of values behind the loads, chunks took 711 us instead of 742, frames 311 instead of 334)
            auto entry_at = [&](int key) -> int { return key < kend ? *(const volatile int32_t *) (table + (key >> pool.page_shift)) : -1; };
            uint4 raw[NG], next[NG];                            // this block's row and the next one's
            // their scales (vd, K warps: those of the value, for the masks)
            uint32_t d[NG], dn[NG], vd[NG], vdn[NG];
            int entry = entry_at(k0 + kt), heldn = -1;          // table entry of the block to be loaded; page of the one in `next`
            auto load = [&](int j) {
                const int key = k0 + j * BLK + kt;
                const int page = (uint32_t) entry < (uint32_t) n_pages ? entry : -1;
                heldn = page;
                // (a row without a page loads page 0's, and its scales become 0 at its use)
                const uint4 * q = (const uint4 *) (q_head + (uint64_t) (uint32_t) max(page, 0) * q_page + (key & pmask) * 16 * NG);
                const uint16_t * s = d_head + (uint64_t) (uint32_t) max(page, 0) * (2 * d_plane) + (key & pmask);
#pragma unroll
                for (int i = 0; i < NG; i++) next[i] = q[i];
#pragma unroll
                for (int i = 0; i < NG; i++) { dn[i] = s[i * P]; vdn[i] = s[(keys ? d_plane : 0) + i * P]; }
                if (j + 1 < nb_all) entry = entry_at(key + BLK);
            };
            if (nb_all > 0) load(0);
            cta_sync();                         // the queries have left the stages' memory
            bool ok = true;
            for (int j = 0; j < nb_all; j++) {
                const int s = j % STAGES, slot = j % SLOTS;
                const bool live = heldn >= 0, hole = !live && k0 + j * BLK + kt < kend;
#pragma unroll
                for (int i = 0; i < NG; i++) { raw[i] = next[i]; d[i] = live ? dn[i] : 0; vd[i] = live ? vdn[i] : 0; }
                if (j + 1 < nb_all) load(j + 1);
                // block j - STAGES, which had this stage, is done with in every tile that took it
                if (j >= STAGES) {
                    const uint32_t ph = (uint32_t) (j / STAGES - 1) & 1u;
                    uint64_t (&empty)[2][STAGES] = keys ? bars.k_empty : bars.v_empty;
                    if (j - STAGES < nb0) ok = warp_wait(a, &empty[0][s], ph, 41);
                    // Where tile 0 has no block j - STAGES, tile 1 alone would set the pace, and this block's masks could take
                    // the place of tile 0's last ones before its softmax has read them: wait for tile 0's last product.
                    else if (keys && j - STAGES == nb0 && nb0 > 0) ok = warp_wait(a, &bars.o_done[0][(nb0 - 1) % NB], (uint32_t) ((nb0 - 1) / NB) & 1u, 40);
                    if (ok && n_tiles == 2) ok = warp_wait(a, &empty[1][s], ph, 42);
                    if (!ok) break;
                }
                if (keys) {
                    const uint32_t holes = __ballot_sync(0xffffffffu, hole);
                    uint32_t any = holes;
#pragma unroll
                    for (int i = 0; i < NG; i++) {
                        const uint32_t m = __ballot_sync(0xffffffffu, not_finite(vd[i]));
                        any |= m;
                        if (lane == 0) s_bad[slot][i][cw] = m;
                    }
                    if (lane == 0) { s_hole[slot][cw] = holes; s_any[slot][cw] = any; }
                } else {
#pragma unroll
                    for (int i = 0; i < NG; i++) {
                        if (not_finite(d[i])) d[i] = 0;
                    }
                }
                const uint32_t dst = (keys ? sK : sV) + s * AT * ATOM + kt * 128;
#pragma unroll
                for (int i = 0; i < W; i++) {
                    const uint4 & q4 = raw[i / 4];
                    const uint32_t w = (i & 3) == 0 ? q4.x : (i & 3) == 1 ? q4.y : (i & 3) == 2 ? q4.z : q4.w;
                    const __half2 d2 = u2h((keys ? d[i % NG] : d[i / 4]) * 0x10001u);     // a key row's groups take turns
                    __half2 x[4];
                    codes4(w, x);
                    st_shared16(dst + (i / 8) * ATOM + (((i & 7) ^ (kt & 7)) << 4), h2u(__hmul2(x[0], d2)), h2u(__hmul2(x[1], d2)),
                                h2u(__hmul2(x[2], d2)), h2u(__hmul2(x[3], d2)));
                }
                fence_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(keys ? &bars.k_full[s] : &bars.v_full[s]);
            }
            if (!ok) abort_sh = 1;
        } else if (warp >= SOFT + CONV) {
            // ---- products of tile t: the whole warp waits, one lane issues
            cta_sync();                         // the queries are in place
            const int t = warp - SOFT - CONV, nb = t == 0 ? nb0 : t < n_tiles ? nb_all : 0;
            const uint32_t q_desc = (uint32_t) sw128_desc(sQ + t * AT * QATOM), k_desc = (uint32_t) sw128_desc(sK), v_desc = (uint32_t) mn_desc(sV), hi = (uint32_t) (sw128_desc(0) >> 32);
            const uint32_t od = tmem + HD * t, qd = tmem + Q_COL + HD / 2 * t, sd = tmem + S_COL + NB * BLK * t;
            auto scores_of = [&](int j) -> bool {
                const int s = j % STAGES;
                if (!warp_wait(a, &bars.k_full[s], (uint32_t) (j / STAGES) & 1u, 43)) return false;
                fence_after();
                const uint32_t id = idesc((min(BLK, kend - k0 - j * BLK) + 15) & ~15, false), ds = sd + BLK * (j % NB);
                const uint32_t k_lo = k_desc + s * (AT * ATOM >> 4);
                if (elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < HD / 16; kk++) {
                        const uint32_t kl = k_lo + ((kk / 4) * ATOM + (kk % 4) * 32 >> 4);
                        if (QT) mma_ts(ds, qd + 8 * kk, kl, hi, id, kk != 0);
                        else mma_ss(ds, q_desc + ((kk / 4) * QATOM + (kk % 4) * 32 >> 4), hi, kl, hi, id, kk != 0);
                    }
                    mma_commit(&bars.s_full[t][j % NB]);
                    mma_commit(&bars.k_empty[t][s]);
                }
                __syncwarp();
                return true;
            };
            bool ok = true;
            for (int j = 0; j < NB && j < nb && ok; j++) ok = scores_of(j);
            for (int j = 0; j < nb && ok; j++) {
                const int s = j % STAGES;
                ok = warp_wait(a, &bars.p_full[t][j % NB], (uint32_t) (j / NB) & 1u, 44) && warp_wait(a, &bars.v_full[s], (uint32_t) (j / STAGES) & 1u, 45);
                if (!ok) break;
                fence_after();
                const int steps = (min(BLK, kend - k0 - j * BLK) + 15) / 16;
                const uint32_t v_lo = v_desc + s * (AT * ATOM >> 4), pa = sd + BLK * (j % NB);
                if (elect_one()) {
                    mma_ts(od, pa, v_lo, hi, idesc(HD, true), j != 0);
#pragma unroll
                    for (int kk = 1; kk < BLK / 16; kk++) {
                        if (kk < steps) mma_ts(od, pa + 8u * kk, v_lo + (kk * 2048 >> 4), hi, idesc(HD, true), 1);
                    }
                    mma_commit(&bars.o_done[t][j % NB]);
                    mma_commit(&bars.v_empty[t][s]);
                }
                __syncwarp();
                // the buffer's next scores go over P_t(j): only when its product is done
                if (j + NB < nb) ok = warp_wait(a, &bars.o_done[t][j % NB], (uint32_t) (j / NB) & 1u, 46) && scores_of(j + NB);
            }
            // the last arrivals of the commits, so that none meets a barrier that is set up anew
            for (int s = 0; s < STAGES && ok; s++) {
                const int n = (nb + STAGES - 1 - s) / STAGES;
                if (n > 0) ok = warp_wait(a, &bars.k_empty[t][s], (uint32_t) (n - 1) & 1u, 50) && warp_wait(a, &bars.v_empty[t][s], (uint32_t) (n - 1) & 1u, 51);
            }
            if (!ok) {
                // the products under way read shared memory and write tensor memory, both about to be given up
                abort_sh = 1;
                if (elect_one()) mma_commit(&bars.drained[t]);
                __syncwarp();
                mbar_wait(&bars.drained[t], 0, 52, &g_kv4_failures.code);
                __syncwarp();
            }
        } else if (128 * (warp >> 2) + 32 * (warp & 3) < cols) {
            // ---- softmax: thread = row
            cta_sync();
            const int t = warp >> 2, nb = t == 0 ? nb0 : nb_all;
            const uint32_t lanes = (uint32_t) (32 * (warp & 3)) << 16;
            const uint32_t ts = tmem + lanes + S_COL + NB * BLK * t, to = tmem + lanes + HD * t;
            float z = col < n_cols ? -FLT_MAX : 0.0f, l = 0.0f;     // about the running maximum less 6 (a whole number), the sum of weights 2^(s - z)
            uint32_t poison = 0;
            bool ok = true, plain = false;
            // O_t += P_t V of block j is done (a warp that asks has seen S(j) or S(j + 1), so block j - NB's is)
            auto product_done = [&](int j, int code) -> bool { return warp_wait(a, &bars.o_done[t][j % NB], (uint32_t) (j / NB) & 1u, code); };
            // Raises z of the rows whose largest s - z of a block is `top` > 14.5 (z is a whole number, and so is the step:
            // sums and O take an exact power of two); returns the step.
            auto raise = [&](float top, int j) -> float {
                float n = 0.0f;
                if (top > 14.5f) n = fabsf(z + top) > 0x1p20f ? top : floorf(top) - 6.0f;
                const float down = ex2(-n);
                z += n;
                l *= down;
                if (j > 0) ok = product_done(j - 1, 48);
                if (j > 0 && ok) {              // O holds the blocks before this one
                    fence_after();
#pragma unroll 1
                    for (int i = 0; i < 2 * NG; i++) {
                        uint32_t y[16];
                        tmem_ld16(to + 16u * i, y);
#pragma unroll
                        for (int k = 0; k < 16; k++) y[k] = __float_as_uint(__uint_as_float(y[k]) * down);
                        tmem_st16(to + 16u * i, y);
                    }
                }
                return n;
            };
            for (int j = 0; j < nb && ok; j++) {
                const int key = k0 + j * BLK;
                const uint32_t tb = ts + BLK * (j % NB);
                if (!warp_wait(a, &bars.s_full[t][j % NB], (uint32_t) (j / NB) & 1u, 47)) { ok = false; break; }
                fence_after();
                uint32_t x[2][32];
                tmem_ld32_async(tb, x[0]);
                tmem_ld32_async(tb + 32u, x[1]);
                const uint2 any = *(const uint2 *) s_any[j % SLOTS];
                const bool odd = (any.x | any.y) != 0;
                const bool whole = __all_sync(0xffffffffu, col >= n_cols || lim >= key + BLK) && !odd;
                if (odd) {
                    for (int c = 0; c < 2; c++) {
#pragma unroll
                        for (int i = 0; i < NG; i++) poison |= (s_bad[j % SLOTS][i][c] & seen(lim - key - 32 * c) & ~s_hole[j % SLOTS][c]) ? 1u << i : 0u;
                    }
                }
                tmem_ld_wait(x[0]);
                tmem_ld_wait(x[1]);
                if (!whole) {                   // scores that the row does not see
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        uint32_t m = seen(lim - key - 32 * h);
                        if (odd) m &= ~s_hole[j % SLOTS][h];
#pragma unroll
                        for (int i = 0; i < 32; i++) {
                            if (!((m >> i) & 1)) x[h][i] = 0xff800000u;
                        }
                    }
                }
                auto largest = [&]() -> float {
                    float mq[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) mq[i] = fmaxf(__uint_as_float(x[0][i]), __uint_as_float(x[1][i]));
#pragma unroll
                    for (int i = 8; i < 32; i += 8) {
#pragma unroll
                        for (int k = 0; k < 8; k++) mq[k] = fmaxf(mq[k], fmaxf(__uint_as_float(x[0][i + k]), __uint_as_float(x[1][i + k])));
                    }
                    return fmaxf(fmaxf(fmaxf(mq[0], mq[1]), fmaxf(mq[2], mq[3])), fmaxf(fmaxf(mq[4], mq[5]), fmaxf(mq[6], mq[7])));
                };
                // One fused step s f - z, where every row of the warp has a z, within 2^20. Beyond that it would differ from the
                // difference of the rounded s f and z by more than 2^-4: there the product is rounded first, and z is a
                // rounded product itself.
                if (!plain) {
                    if (z == -FLT_MAX) {        // a row that has seen nothing so far
                        const float mx = largest();
                        if (mx != -INFINITY) z = fabsf(mx * f) > 0x1p20f ? mx * f : floorf(mx * f) - 6.0f;
                    }
                    plain = __all_sync(0xffffffffu, fabsf(z) <= 0x1p20f);
                }
                if (plain) {
                    const uint64_t f2 = pack2(f, f), z2 = pack2(-z, -z);
#pragma unroll
                    for (int i = 0; i < 32; i++) {
                        uint32_t & a0 = x[i / 16][2 * (i % 16)], & a1 = x[i / 16][2 * (i % 16) + 1];
                        const float2 v = unpack2(fma2(pack2(__uint_as_float(a0), __uint_as_float(a1)), f2, z2));
                        a0 = __float_as_uint(v.x);
                        a1 = __float_as_uint(v.y);
                    }
                } else {
#pragma unroll 1
                    for (int h = 0; h < 2; h++) {
#pragma unroll
                        for (int i = 0; i < 32; i++) {
                            const float v = __fadd_rn(__fmul_rn(__uint_as_float(x[0][i]), f), -z);
                            x[0][i] = x[1][i];
                            x[1][i] = __float_as_uint(v);
                        }
                    }
                }
                const float top = largest();
                if (__any_sync(0xffffffffu, top > 14.5f)) {
                    const float n = raise(top, j);
                    if (!ok) break;
                    plain = __all_sync(0xffffffffu, fabsf(z) <= 0x1p20f);
#pragma unroll
                    for (int i = 0; i < 32; i++) {
                        x[0][i] = __float_as_uint(__uint_as_float(x[0][i]) - n);
                        x[1][i] = __float_as_uint(__uint_as_float(x[1][i]) - n);
                    }
                }
                uint64_t sum2[4] = {0, 0, 0, 0};
#pragma unroll
                for (int h = 0; h < 2; h++) {
#pragma unroll
                    for (int i = 0; i < 32; i++) x[h][i] = __float_as_uint(ex2(__uint_as_float(x[h][i])));
                }
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t p[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const float p0 = __uint_as_float(x[h][2 * i]), p1 = __uint_as_float(x[h][2 * i + 1]);
                        sum2[i & 3] = add2(sum2[i & 3], pack2(p0, p1));
                        p[i] = pack_h2(p0, p1);
                    }
                    tmem_st16(tb + 16u * h, p);
                }
                const float2 sa = unpack2(add2(add2(sum2[0], sum2[1]), add2(sum2[2], sum2[3])));
                l += sa.x + sa.y;
                tmem_wait_st();
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars.p_full[t][j % NB]);
            }
            if (ok && nb > 0) ok = product_done(nb - 1, 49);
            if (!ok) abort_sh = 1;
            fence_after();
            const bool there = col < n_cols;
            const float inv = used > 1 ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
            const size_t at = ((size_t) blockIdx.x * a.n_rows + row) * a.heads + head;
            T * out = (T *) a.out + (long long) row * a.o_tok + head * a.o_head;
#pragma unroll 1
            for (int i = 0; i < NG; i++) {
                uint32_t x[32];
                if (ok && nb > 0) {             // (the whole warp agrees)
                    tmem_ld32_async(to + 32u * i, x);
                    tmem_ld_wait(x);
                } else {
#pragma unroll
                    for (int k = 0; k < 32; k++) x[k] = 0u;
                }
                if (there) {
                    const bool nan = ((poison >> i) & 1) || !ok;
#pragma unroll
                    for (int w = 0; w < 4; w++) {   // columns 8 w + 2 c + e hold channels 8 w + c + 4 e
                        float y[8];
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            y[c] = nan ? __int_as_float(0x7fffffff) : __uint_as_float(x[8 * w + 2 * c]) * inv;
                            y[c + 4] = nan ? __int_as_float(0x7fffffff) : __uint_as_float(x[8 * w + 2 * c + 1]) * inv;
                        }
                        if (used > 1) {
                            float4 * d = (float4 *) (sp.o + at * HD + 32 * i + 8 * w);
                            d[0] = make_float4(y[0], y[1], y[2], y[3]);
                            d[1] = make_float4(y[4], y[5], y[6], y[7]);
                        } else {
                            T e[8];
#pragma unroll
                            for (int c = 0; c < 8; c++) e[c] = to_type<T>(y[c]);
                            T * d = out + 32 * i + 8 * w;
                            if (vec & 4) {
                                *(uint4 *) d = *(const uint4 *) e;
                            } else {
#pragma unroll
                                for (int c = 0; c < 8; c++) d[c] = e[c];
                            }
                        }
                    }
                }
                __syncwarp();
            }
            if (there && used > 1) sp.ml[at] = make_float2(z, l);
        }
        else {
            cta_sync();                         // a softmax warp without rows
        }
        cta_sync();
        if (*(volatile int *) &abort_sh) {
            if (threadIdx.x == 0) atomicAdd(&g_kv4_failures.count, 1u);
            // the columns that this CTA would have come to: not numbers either
            for (c0 += tiles * 256; c0 < n_cols; c0 += tiles * 256) {
                for (int i = threadIdx.x; i < min(256, n_cols - c0) * HD; i += THREADS) {
                    const int col = c0 + i / HD, row = rq.row0 + col / G, head = kh * G + col % G;
                    const size_t at = ((size_t) blockIdx.x * a.n_rows + row) * a.heads + head;
                    if (used <= 1) ((T *) a.out)[(long long) row * a.o_tok + head * a.o_head + i % HD] = to_type<T>(__int_as_float(0x7fffffff));
                    else sp.o[at * HD + i % HD] = __int_as_float(0x7fffffff);
                    if (used > 1 && i % HD == 0) sp.ml[at] = make_float2(-FLT_MAX, 0.0f);
                }
            }
            break;
        }
        if (threadIdx.x == 0) {                 // the next columns start with fresh barriers
            for (int i = 0; i < (int) (sizeof(Bars) / 8); i++) {
                asm volatile("mbarrier.inval.shared::cta.b64 [%0];" :: "r"(smem_u32((uint64_t *) &bars + i)) : "memory");
            }
        }
        __syncthreads();
    }
    if (warp == SOFT) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem_sh), "r"(512) : "memory");
    }
}

template <class T, int NG>
int launch(const Kv4Pool & p, const Args & a, const Split & sp, int tiles, int vec, cudaStream_t st) {
    if (allow_smem<k_kv4_tiles<T, NG>>((int) tiles_smem<NG>())) return -1;
    const dim3 grid((unsigned) sp.n_split, (unsigned) (p.heads * tiles), (unsigned) a.n_req);
    JB_CUDA(launch_pdl(k_kv4_tiles<T, NG>, grid, dim3(THREADS), tiles_smem<NG>(), st, p, a, sp, tiles, vec));
    return 0;
}

template <class T>
int launch_dim(const Kv4Pool & p, const Args & a, const Split & sp, int tiles, int vec, cudaStream_t st) {
    switch (p.hd / 32) {
        case 1: return launch<T, 1>(p, a, sp, tiles, vec, st);
        case 2: return launch<T, 2>(p, a, sp, tiles, vec, st);
        case 3: return launch<T, 3>(p, a, sp, tiles, vec, st);
        default: return launch<T, 4>(p, a, sp, tiles, vec, st);
    }
}

}  // namespace

int kv4_error_flag(cudaStream_t st) {
    constexpr int DEVICES = 256;
    static std::atomic<unsigned> told[DEVICES];
    int dev = 0;
    Kv4Failures v = {0, 0};
    if (!cuda_ok(cudaGetDevice(&dev), "reading the 4-bit cache's failures") || dev >= DEVICES ||
        !cuda_ok(cudaMemcpyFromSymbolAsync(&v, g_kv4_failures, sizeof(v), 0, cudaMemcpyDeviceToHost, st), "reading the 4-bit cache's failures") ||
        !cuda_ok(cudaStreamSynchronize(st), "reading the 4-bit cache's failures")) {
        return -1;
    }
    unsigned last = told[dev].load();
    while ((int) (v.count - last) > 0) {                     // (another thread may have told a later count)
        if (told[dev].compare_exchange_weak(last, v.count)) return v.code;
    }
    return 0;
}

int kv4_tiles(const Kv4Pool & p, const Kv4Attn & attn, const Kv4Waits & waits, const Split & sp, int tiles, int vec, cudaStream_t st) {
    const Args a{attn, waits};
    return a.type == KV4_F16 ? launch_dim<__half>(p, a, sp, tiles, vec, st) : launch_dim<__nv_bfloat16>(p, a, sp, tiles, vec, st);
}

}  // namespace jb
