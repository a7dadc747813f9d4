// Attention over the paged 4-bit cache for many rows (kv4.h; the formula is in kv4_attention.cu): tcgen05 products.
//
// One CTA per (request, cache head, 256 columns, range of keys); a column is a (new token, head of the group) pair, a
// row of the two 128-row tiles here. Keys come in blocks of 128. Warps:
//   0 .. 7   softmax: one thread per row (4 warps a tile, one per TMEM lane quadrant). They write the queries into shared
//            memory once (scaled by a power of two into f16's range), then per block read their row of S = Q K^T from
//            TMEM twice (its maximum, then the weights), and put P = 2^(s - m + 10) back in f16 over the front half of S's
//            columns, where the second product takes it as its A operand: P never passes through shared memory.
//            O stays in TMEM; it is rescaled only when a row's maximum rises by more than 2^4 (P <= 2^14 fits f16).
//   8 .. 11  conversion: one thread per key, K and V rows from 4 bits to d (c - 8) in f16 (exact, kv4.h), written
//            in the 128-byte swizzle of the products' operands (K: K-major; V: MN-major, keys down the rows).
//            The next block's codes are loaded before this one's are converted.
//   12       one lane issues the products: S_t = Q_t K^T (M 128, N 128), O_t += P_t V (M 128, N hd), the tiles in turn,
//            so that one tile's products run under the other's softmax.
// Within 8 channels the operands keep the order in which codes unpack, 0 4 1 5 2 6 3 7: Q is written in the order of
// K's words, O's columns are put right when they are stored.
// TMEM: S of tile t at column 128 t, O of tile t at 256 + 128 t.
// A value scale that is not finite enters as zeros; the rows that see such a key get NaN in that group at the end, so a NaN
// behind a row's mask does not reach it (0 * NaN).
// Every mbarrier wait is bounded: on a timeout the kernel raises the error flag, its rows become NaN, and it ends.
#include "kv4_device.h"
#include "common.h"
#include "launch.h"
#include "tcgen05.cuh"

#include <cfloat>

namespace jb {

__device__ int g_kv4_error = 0;

namespace {

using namespace tc;

constexpr int BLK = 128;                        // keys per block
constexpr int SOFT = 8, CONV = 4;               // warps of each kind
constexpr int THREADS = 32 * (SOFT + CONV + 1);
constexpr uint32_t ATOM = 128 * 128;            // bytes of 128 rows x 64 f16

__host__ __device__ constexpr uint32_t idesc(int n, bool b_mn_major) {      // kind::f16, f16 in, f32 out, M 128
    return (1u << 4) | ((uint32_t) (n >> 3) << 17) | ((uint32_t) (128 >> 4) << 24) | (b_mn_major ? 1u << 16 : 0u);
}
// MN-major operand in the 128-byte swizzle: 64-element columns of atoms one block of rows (ATOM bytes) apart (LBO),
// 8-row groups 1024 bytes apart (SBO)
__device__ __forceinline__ uint64_t mn_desc(uint32_t saddr) {
    uint64_t d = sw128_desc(saddr) & ~((uint64_t) 0x3FFF << 16);
    return d | (uint64_t) (ATOM >> 4) << 16;
}
// D += A B with A in tensor memory
__device__ __forceinline__ void mma_f16_ta(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        :: "r"(d), "r"(a), "l"(b), "r"(id), "r"(acc));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        :: "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
           "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    uint32_t a[16], b[16];
#pragma unroll
    for (int i = 0; i < 16; i++) { a[i] = r[i]; b[i] = r[16 + i]; }
    tmem_st16(taddr, a);
    tmem_st16(taddr + 16, b);
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

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

// the whole warp waits, and agrees on the outcome
__device__ __forceinline__ bool warp_wait(uint64_t * bar, uint32_t parity, int code) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, code, &g_kv4_error));
}
__device__ __forceinline__ bool aborted(const int * flag) { return __any_sync(0xffffffffu, *(const volatile int *) flag != 0); }

constexpr int SLOTS = 4;        // blocks whose key masks are kept (a block's is rewritten when both tiles are done with it)

template <int NG> __host__ __device__ constexpr int atoms() { return (NG + 1) / 2; }
template <int NG> constexpr size_t tiles_smem() { return (size_t) atoms<NG>() * ATOM * 6 + 1024; }   // Q x 2, K x 2, V x 2

template <class T, int NG>
__global__ void __launch_bounds__(THREADS, 1) k_kv4_tiles(const Kv4Pool pool, const Kv4Attn a, const Split sp, int tiles, int vec) {
    constexpr int HD = 32 * NG, AT = atoms<NG>(), W = 4 * NG;      // W: 8-channel words of a row
    extern __shared__ uint8_t smem_raw[];
    uint8_t * sQ = (uint8_t *) (((uintptr_t) smem_raw + 1023) & ~(uintptr_t) 1023);
    uint8_t * sK = sQ + 2 * AT * ATOM, * sV = sK + 2 * AT * ATOM;
    __shared__ __align__(8) uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_done[2];
    // per block and 32 keys: any exception; keys without a page; keys whose value scale of a group is not finite
    __shared__ __align__(16) uint32_t s_any[SLOTS][4], s_hole[SLOTS][4], s_bad[SLOTS][NG][4];
    __shared__ uint32_t tmem_sh;
    __shared__ int abort_sh;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kh = blockIdx.y / tiles, r = blockIdx.z, G = a.heads / pool.heads;
    const Req rq = request_of(a, pool.page_shift, r);
    const int n_cols = (rq.row1 - rq.row0) * G;
    const int span = sp.span(rq.len), used = sp.used(rq.len);
    const int k0 = blockIdx.x * span;
    if (n_cols <= 0 || (int) (blockIdx.y % tiles) * 256 >= n_cols || (blockIdx.x && (int) blockIdx.x >= used)) return;

    if (warp == SOFT + CONV) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(&tmem_sh)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (threadIdx.x == 0) abort_sh = 0;

    for (int c0 = (int) (blockIdx.y % tiles) * 256; c0 < n_cols; c0 += tiles * 256) {
        const int cols = min(256, n_cols - c0), n_tiles = cols > 128 ? 2 : 1;
        const int kend = min(visible(rq, rq.row0 + (c0 + cols - 1) / G, a.frame), min(rq.len, k0 + span));   // the last row sees most
        const int nb_all = kend > k0 ? (kend - k0 + BLK - 1) / BLK : 0;
        const int kend0 = n_tiles == 1 ? kend : min(visible(rq, rq.row0 + (c0 + 127) / G, a.frame), kend);
        const int nb0 = kend0 > k0 ? (kend0 - k0 + BLK - 1) / BLK : 0;          // blocks of tile 0
        if (threadIdx.x == 0) {
            for (int s = 0; s < 2; s++) {
                mbar_init(&k_full[s], CONV); mbar_init(&k_empty[s], 1);
                mbar_init(&v_full[s], CONV); mbar_init(&v_empty[s], 1);
                mbar_init(&s_full[s], 1); mbar_init(&o_done[s], 1);
                mbar_init(&p_full[s], (uint32_t) max(1, (min(128, cols - 128 * s) + 31) / 32));
            }
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        // ---- queries: thread = row of the tiles, words in the order of the key rows
        float f = 0.0f;                         // of this row's scores, in log2 units
        int lim = 0;                            // keys this row sees
        const int col = c0 + threadIdx.x;
        const int row = rq.row0 + (warp < SOFT && col < n_cols ? col / G : 0), head = kh * G + (col < n_cols ? col % G : 0);
        if (warp < SOFT) {
            const bool there = col < n_cols;
            const T * q = (const T *) a.q + (long long) row * a.q_tok + head * a.q_head;
            auto word = [&](int s, float (&x)[8]) {
                const T * p = q + 32 * (s % NG) + 8 * (s / NG);
                T e[8];
                if (!there) {
#pragma unroll
                    for (int c = 0; c < 8; c++) e[c] = to_type<T>(0.0f);
                } else if (vec & 1) {
                    *(uint4 *) e = *(const uint4 *) p;
                } else {
#pragma unroll
                    for (int c = 0; c < 8; c++) e[c] = p[c];
                }
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
            f = fabsf(a.scale) * 1.4426950408889634f * __int_as_float((127 - ex) << 23);
            if (there) lim = min(visible(rq, row, a.frame), kend);
            uint8_t * dst = sQ + (warp >> 2) * AT * ATOM + (threadIdx.x & 127) * 128;
#pragma unroll
            for (int s = 0; s < W; s++) {
                word(s, x);
                uint4 w;
                w.x = pack_h2(x[0] * up, x[4] * up); w.y = pack_h2(x[1] * up, x[5] * up);
                w.z = pack_h2(x[2] * up, x[6] * up); w.w = pack_h2(x[3] * up, x[7] * up);
                *(uint4 *) (dst + (s / 8) * ATOM + (((s & 7) ^ (lane & 7)) << 4)) = w;
            }
            fence_async();
        }
        fence_before();
        __syncthreads();
        fence_after();
        const uint32_t tmem = tmem_sh;

        if (warp >= SOFT && warp < SOFT + CONV) {
            // ---- conversion: thread = key of the block
            const int kt = threadIdx.x - 32 * SOFT, cw = warp - SOFT;
            const int32_t * table = a.table + (size_t) r * a.width;
            const int n_pages = (int) (pool.n_slots >> pool.page_shift), pmask = (1 << pool.page_shift) - 1, P = 1 << pool.page_shift;
            const size_t q_plane = ((size_t) pool.heads << pool.page_shift) * 16 * NG, d_plane = ((size_t) pool.heads * NG) << pool.page_shift;
            auto page_at = [&](int key) -> int {
                const int p = key < kend ? __ldg(table + (key >> pool.page_shift)) : -1;
                return p < n_pages ? p : -1;
            };
            uint4 kr[NG], vr[NG], kn[NG], vn[NG];               // this block's rows and the next one's
            __half kd[NG], vd[NG], kdn[NG], vdn[NG];
            int page = page_at(k0 + kt), held = -1, heldn = -1;     // of the block to be loaded; of those in registers
            auto load = [&](int j) {
                const int key = k0 + j * BLK + kt;
                heldn = page;
                if (page >= 0) {
                    const size_t qa = kv4_q_at(pool, page, 0, kh, key & pmask), da = kv4_d_at(pool, page, 0, kh, key & pmask);
                    const uint4 * q = (const uint4 *) (pool.q + qa);
                    const uint4 * v = (const uint4 *) (pool.q + qa + q_plane);
#pragma unroll
                    for (int i = 0; i < NG; i++) { kn[i] = q[i]; vn[i] = v[i]; }
#pragma unroll
                    for (int i = 0; i < NG; i++) { kdn[i] = pool.d[da + (size_t) i * P]; vdn[i] = pool.d[da + d_plane + (size_t) i * P]; }
                } else {
#pragma unroll
                    for (int i = 0; i < NG; i++) { kn[i] = vn[i] = make_uint4(0, 0, 0, 0); kdn[i] = vdn[i] = __ushort_as_half(0); }
                }
                if (j + 1 < nb_all) page = page_at(key + BLK);
            };
            if (nb_all > 0) load(0);
            bool ok = true;
            for (int j = 0; j < nb_all; j++) {
                const int s = j & 1, u = j >> 1;
                held = heldn;
#pragma unroll
                for (int i = 0; i < NG; i++) { kr[i] = kn[i]; vr[i] = vn[i]; kd[i] = kdn[i]; vd[i] = vdn[i]; }
                if (j + 1 < nb_all) load(j + 1);
                const bool live = held >= 0;
                // one operand row: the words of w, scaled by their groups, at row kt of a block of atoms
                auto convert = [&](uint8_t * dst, const uint4 (&raw)[NG], const __half (&d)[NG], bool keys) {
#pragma unroll
                    for (int i = 0; i < W; i++) {
                        const uint4 & q4 = raw[i / 4];
                        const uint32_t w = (i & 3) == 0 ? q4.x : (i & 3) == 1 ? q4.y : (i & 3) == 2 ? q4.z : q4.w;
                        const __half2 d2 = __half2half2(d[keys ? i % NG : i / 4]);
                        __half2 x[4];
                        codes4(w, x);
                        uint4 o;
                        o.x = h2u(__hmul2(x[0], d2)); o.y = h2u(__hmul2(x[1], d2)); o.z = h2u(__hmul2(x[2], d2)); o.w = h2u(__hmul2(x[3], d2));
                        *(uint4 *) (dst + (i / 8) * ATOM + kt * 128 + (((i & 7) ^ (kt & 7)) << 4)) = o;
                    }
                };
                if (u >= 1 && !warp_wait(&k_empty[s], (uint32_t) (u - 1) & 1u, 41)) { ok = false; break; }
                if (aborted(&abort_sh)) { ok = false; break; }
                const uint32_t hole = __ballot_sync(0xffffffffu, !live && k0 + j * BLK + kt < kend);
                uint32_t any = hole;
#pragma unroll
                for (int i = 0; i < NG; i++) {
                    const bool bad = __hisnan(vd[i]) || __hisinf(vd[i]);
                    const uint32_t m = __ballot_sync(0xffffffffu, bad);
                    if (bad) vd[i] = __ushort_as_half(0);
                    any |= m;
                    if (lane == 0) s_bad[j % SLOTS][i][cw] = m;
                }
                if (lane == 0) { s_hole[j % SLOTS][cw] = hole; s_any[j % SLOTS][cw] = any; }
                convert(sK + s * AT * ATOM, kr, kd, true);
                fence_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&k_full[s]);
                if (u >= 1 && !warp_wait(&v_empty[s], (uint32_t) (u - 1) & 1u, 42)) { ok = false; break; }
                convert(sV + s * AT * ATOM, vr, vd, false);
                fence_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&v_full[s]);
            }
            if (!ok) abort_sh = 1;
        } else if (warp == SOFT + CONV) {
            // ---- products: one lane
            if (lane == 0 && nb_all > 0) {
                const uint32_t q_u = smem_u32(sQ), k_u = smem_u32(sK), v_u = smem_u32(sV);
                bool ok = true;
                auto issue_s = [&](int t, int j) {
                    const uint32_t id = idesc((min(BLK, kend - k0 - j * BLK) + 15) & ~15, false);
                    const uint32_t qa = q_u + t * AT * ATOM, ka = k_u + (j & 1) * AT * ATOM;
#pragma unroll
                    for (int kk = 0; kk < HD / 16; kk++) {
                        const uint32_t o = (kk / 4) * ATOM + (kk % 4) * 32;
                        mma_kind_f16(tmem + 128u * t, sw128_desc(qa + o), sw128_desc(ka + o), id, kk != 0);
                    }
                    mma_commit(&s_full[t]);
                };
                ok = mbar_wait(&k_full[0], 0, 43, &g_kv4_error);
                fence_after();
                if (ok) {
                    if (nb0 > 0) issue_s(0, 0);
                    if (n_tiles == 2) issue_s(1, 0);
                    mma_commit(&k_empty[0]);
                }
                for (int j = 0; j < nb_all && ok; j++) {
                    const int s = j & 1;
                    const uint32_t ph = (uint32_t) (j >> 1) & 1u;
                    ok = mbar_wait(&v_full[s], ph, 44, &g_kv4_error);
                    if (ok && j + 1 < nb_all) ok = mbar_wait(&k_full[s ^ 1], (uint32_t) ((j + 1) >> 1) & 1u, 45, &g_kv4_error);
                    const int steps = (min(BLK, kend - k0 - j * BLK) + 15) / 16;
                    for (int t = 0; t < n_tiles && ok; t++) {
                        const int nb = t == 0 ? nb0 : nb_all;
                        if (j >= nb) continue;
                        ok = mbar_wait(&p_full[t], (uint32_t) j & 1u, 46, &g_kv4_error);
                        if (!ok) break;
                        fence_after();
                        const uint32_t va = v_u + s * AT * ATOM;
                        for (int kk = 0; kk < steps; kk++) {
                            mma_f16_ta(tmem + 256u + 128u * t, tmem + 128u * t + 8u * kk, mn_desc(va + kk * 2048), idesc(HD, true), j != 0 || kk != 0);
                        }
                        mma_commit(&o_done[t]);
                        if (j + 1 < nb) issue_s(t, j + 1);
                    }
                    if (!ok) break;
                    mma_commit(&v_empty[s]);
                    if (j + 1 < nb_all) mma_commit(&k_empty[s ^ 1]);
                }
                // the last arrivals of the commits, so that none meets a barrier that is set up anew
                for (int s = 0; s < 2 && ok; s++) {
                    const int n = (nb_all + 1 - s) / 2;
                    if (n > 0) ok = mbar_wait(&k_empty[s], (uint32_t) (n - 1) & 1u, 50, &g_kv4_error) && mbar_wait(&v_empty[s], (uint32_t) (n - 1) & 1u, 51, &g_kv4_error);
                }
                if (!ok) abort_sh = 1;
            }
            __syncwarp();
        } else if (128 * (warp >> 2) + 32 * (warp & 3) < cols) {
            // ---- softmax: thread = row
            const int t = warp >> 2, nb = t == 0 ? nb0 : nb_all;
            const uint32_t lanes = (uint32_t) (32 * (warp & 3)) << 16;
            const uint32_t ts = tmem + lanes + 128u * t, to = tmem + lanes + 256u + 128u * t;
            float z = -FLT_MAX, l = 0.0f;       // the running maximum less 10, the sum of weights 2^(s - z)
            uint32_t poison = 0;
            bool ok = true;
            for (int j = 0; j < nb; j++) {
                const int key = k0 + j * BLK, nc = (min(BLK, kend - key) + 31) / 32;
                if (!warp_wait(&s_full[t], (uint32_t) j & 1u, 47)) { ok = false; break; }
                fence_after();
                const uint4 any = *(const uint4 *) s_any[j % SLOTS];
                const bool odd = (any.x | any.y | any.z | any.w) != 0;
                const bool whole = __all_sync(0xffffffffu, col >= n_cols || lim >= key + 32 * nc) && !odd;
                uint32_t see[4];                // keys of the block that this row sees, in the block's columns
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const int n = lim - key - 32 * c;
                    see[c] = n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
                }
                if (odd) {
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        see[c] &= ~s_hole[j % SLOTS][c];
#pragma unroll
                        for (int i = 0; i < NG; i++) poison |= (s_bad[j % SLOTS][i][c] & see[c]) ? 1u << i : 0u;
                    }
                }
                // maximum
                uint32_t x[32];
                float mx = -INFINITY;
                for (int c = 0; c < nc; c++) {
                    tmem_ld32_async(ts + 32u * c, x);
                    tmem_ld_wait(x);
                    if (!whole) {
                        const uint32_t m = c == 0 ? see[0] : c == 1 ? see[1] : c == 2 ? see[2] : see[3];
#pragma unroll
                        for (int i = 0; i < 32; i++) {
                            if (!((m >> i) & 1)) x[i] = 0xff800000u;
                        }
                    }
                    float mq[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) mq[i] = fmaxf(__uint_as_float(x[i]), __uint_as_float(x[i + 4]));
#pragma unroll
                    for (int i = 8; i < 32; i += 8) {
#pragma unroll
                        for (int k = 0; k < 4; k++) mq[k] = fmaxf(mq[k], fmaxf(__uint_as_float(x[i + k]), __uint_as_float(x[i + k + 4])));
                    }
                    mx = fmaxf(mx, fmaxf(fmaxf(mq[0], mq[1]), fmaxf(mq[2], mq[3])));
                }
                mx = mx == -INFINITY ? mx : mx * f;
                const bool raise = mx - z > 14.0f;
                if (__any_sync(0xffffffffu, raise)) {
                    const float nz = raise ? below(mx) : z, c = nz == z ? 1.0f : ex2(z - nz);
                    z = nz;
                    l *= c;
                    if (j > 0) {                // O holds the blocks before this one
                        if (!warp_wait(&o_done[t], (uint32_t) (j - 1) & 1u, 48)) { ok = false; break; }
                        fence_after();
#pragma unroll 1
                        for (int i = 0; i < NG; i++) {
                            tmem_ld32_async(to + 32u * i, x);
                            tmem_ld_wait(x);
#pragma unroll
                            for (int k = 0; k < 32; k++) x[k] = __float_as_uint(__uint_as_float(x[k]) * c);
                            tmem_st32(to + 32u * i, x);
                        }
                        tmem_wait_st();
                    }
                }
                // weights
                // one fused step s f - z; beyond 2^20 the rounded maximum in z differs from it by more than 2^-4, and the
                // product is rounded first, as the maximum's was, so that the largest weight stays what it should be
                const bool huge = __any_sync(0xffffffffu, fabsf(z) > 0x1p20f && z != -FLT_MAX);
                const uint64_t f2 = pack2(f, f), z2 = pack2(-z, -z);
                uint64_t sum2[2] = {0, 0};
                for (int c = 0; c < nc; c++) {
                    tmem_ld32_async(ts + 32u * c, x);
                    tmem_ld_wait(x);
                    uint32_t p[16];
                    const uint32_t m = whole ? 0xffffffffu : c == 0 ? see[0] : c == 1 ? see[1] : c == 2 ? see[2] : see[3];
                    if (!huge) {
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const float2 y = unpack2(fma2(pack2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), f2, z2));
                            x[2 * i] = __float_as_uint(ex2(y.x));
                            x[2 * i + 1] = __float_as_uint(ex2(y.y));
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; i++) x[i] = __float_as_uint(ex2(__fadd_rn(__fmul_rn(__uint_as_float(x[i]), f), -z)));
                    }
                    if (!whole) {
#pragma unroll
                        for (int i = 0; i < 32; i++) {
                            if (!((m >> i) & 1)) x[i] = 0u;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const float p0 = __uint_as_float(x[2 * i]), p1 = __uint_as_float(x[2 * i + 1]);
                        sum2[i & 1] = add2(sum2[i & 1], pack2(p0, p1));
                        p[i] = pack_h2(p0, p1);
                    }
                    tmem_st16(ts + 16u * c, p);
                }
                const float2 sa = unpack2(add2(sum2[0], sum2[1]));
                l += sa.x + sa.y;
                tmem_wait_st();
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[t]);
                if (aborted(&abort_sh)) { ok = false; break; }
            }
            if (ok && nb > 0) ok = warp_wait(&o_done[t], (uint32_t) (nb - 1) & 1u, 49);
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
        fence_before();
        __syncthreads();
        fence_after();
        if (*(volatile int *) &abort_sh) break;
        if (threadIdx.x == 0) {                 // the next columns start with fresh barriers
            for (int s = 0; s < 2; s++) {
                for (uint64_t * b : {&k_full[s], &k_empty[s], &v_full[s], &v_empty[s], &s_full[s], &p_full[s], &o_done[s]}) {
                    asm volatile("mbarrier.inval.shared::cta.b64 [%0];" :: "r"(smem_u32(b)) : "memory");
                }
            }
        }
        __syncthreads();
    }
    if (warp == SOFT + CONV) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem_sh), "r"(512) : "memory");
    }
}

template <class T, int NG>
int launch(const Kv4Pool & p, const Kv4Attn & a, const Split & sp, int tiles, int vec, cudaStream_t st) {
    JB_CUDA(cudaFuncSetAttribute(k_kv4_tiles<T, NG>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) tiles_smem<NG>()));
    const dim3 grid((unsigned) sp.n_split, (unsigned) (p.heads * tiles), (unsigned) a.n_req);
    JB_CUDA(launch_pdl(k_kv4_tiles<T, NG>, grid, dim3(THREADS), tiles_smem<NG>(), st, p, a, sp, tiles, vec));
    return 0;
}

template <class T>
int launch_dim(const Kv4Pool & p, const Kv4Attn & a, const Split & sp, int tiles, int vec, cudaStream_t st) {
    switch (p.hd / 32) {
        case 1: return launch<T, 1>(p, a, sp, tiles, vec, st);
        case 2: return launch<T, 2>(p, a, sp, tiles, vec, st);
        case 3: return launch<T, 3>(p, a, sp, tiles, vec, st);
        default: return launch<T, 4>(p, a, sp, tiles, vec, st);
    }
}

}  // namespace

int kv4_tiles(const Kv4Pool & p, const Kv4Attn & a, const Split & sp, int tiles, int vec, cudaStream_t st) {
    return a.type == KV4_F16 ? launch_dim<__half>(p, a, sp, tiles, vec, st) : launch_dim<__nv_bfloat16>(p, a, sp, tiles, vec, st);
}

}  // namespace jb
