// Attention over the paged 4-bit cache (kv4.h).
//
//   row i of request r (of n = q_start[r + 1] - q_start[r]) stands at position p = lens[r] - n + i and sees the keys
//   j < lens[r], and with frame > 0 only j < (p / frame + 1) frame (none for p < 0):
//   out = sum_j w_j v_j / sum_j w_j,  w_j = exp(scale q . k_j - max);  0 for a row that sees nothing.
//
// k_kv4_rows, for few rows: one pass over the cache, bound by its 0.5625 bytes a value. The query rows that share a
// cache head (new tokens x the heads of its group) are columns of the products, 8 or 16 of them:
//   S^T [16 keys x 8 rows]  = K [16 x hd] Q^T          mma m16n8k16, one accumulator per 32-channel group: the codes go
//                                                 in as the integers -8 .. 7 (exact in f16), the group's scale
//                                                 multiplies the f32 sum
//   O^T [hd x 8 rows]      += V^T [hd x 16 keys] P^T   the operand is d (c - 8), exact in f16; P = 2^(s - m + 10) in
//                                                 f16: the 2^10 keeps weights down to 2^-24 of the largest
//                                                 normal, the 11 bits cost half an ulp of f16 a weight at most
// Both products take the cache as the A operand, in the order in which it lies in memory: key rows for S^T (a lane's 8
// channels of each group are one 4-byte word), and for O^T a pair of key rows' words merged nibble by nibble; P^T comes
// from S^T by an 8 x 8 transpose inside the warp (movmatrix). Queries are scaled by a power of two per row into f16's
// range (bf16 has 8 more exponent bits than it needs here), which the scores' factor undoes.
// Each warp runs by itself over every fourth step of 32 keys of the CTA's range, fed by its own two-stage cp.async ring
// (the four states are merged at the end); the maximum is raised, and the sums rescaled, only when a score passes it
// by 2^4, so most steps do no reduction across lanes. A long context is split over CTAs, whose partial sums
// k_kv4_merge joins.
#include "kv4_device.h"
#include "common.h"
#include "launch.h"
#include "kprof.h"

#include <algorithm>
#include <cfloat>
#include <type_traits>

namespace jb {

namespace {

// The subtrahend z of a score s in its weight 2^(s - z), for a largest score m: m - 10, so that weights go up to 2^10 (2^14
// before z is raised), within f16; m itself where m - 10 would be rounded (|m| > 2^20), so that s - z <= 0 there.
__device__ __forceinline__ float below(float m) { return fabsf(m) > 0x1p20f ? m : m - 10.0f; }

__device__ __forceinline__ uint32_t smem_addr(const void * p) { return (uint32_t) __cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp_async16(uint32_t dst, const void * src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory"); }

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// d = a b
__device__ __forceinline__ void mma16816_0(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%10, %10, %10, %10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void wait_for_grid() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

constexpr int STEP = 32;        // keys a warp takes at a time
constexpr int STAGES = 2;          // (3: 128 us for 64 sessions of 1000 .. 8190 keys instead of 121)
constexpr int WARPS = 4;

template <int NG> __host__ __device__ constexpr int row_bytes() { return 16 * NG; }
template <int NG> __host__ __device__ constexpr int stage_bytes() { return 2 * STEP * row_bytes<NG>() + 2 * NG * STEP * 2; }
template <int NG, int NT> constexpr int rows_smem() {
    const int ring = WARPS * STAGES * stage_bytes<NG>(), merge = WARPS * 8 * NT * (32 * NG + 4 + 2) * 4;
    return ring > merge ? ring : merge;
}

// Where row r of a step lies in a stage, and the 16-byte chunk c of it: rows 4 .. 7 of each 8 change places pairwise, and
// of four-chunk rows every other pair swaps its halves, so that the reads below (8 lanes of consecutive rows, and 4
// lanes of every other row) touch different banks.
__device__ __forceinline__ int row_pos(int r) { return r ^ ((r >> 2) & 1); }
template <int NG> __device__ __forceinline__ int chunk_pos(int pos, int c) { return NG == 4 ? c ^ (pos & 2) : c; }

template <class T, int NG, int NT>
__global__ void __launch_bounds__(32 * WARPS, NT == 1 ? 4 : 3) k_kv4_rows(const Kv4Pool pool, const Kv4Attn a, const Split sp, int tiles,
                                                                          int vec, int rest) {
    constexpr int HD = 32 * NG, RB = row_bytes<NG>(), SB = stage_bytes<NG>(), MT = 2 * NG;
    // After the tiles kernel (rest) the wait comes last: this grid starts when all of that kernel's CTAs have passed their own
    // wait, so what both read is there, and it runs on the SMs that its last CTAs leave idle; the wait at the
    // end keeps whatever follows behind both.
    if (!rest) wait_for_grid();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ uint32_t s_poison[8 * NT];
    __shared__ int2 s_col[8 * NT];                           // row and head of each column
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int kh = blockIdx.y / tiles, r = blockIdx.z, G = a.heads / pool.heads;
    const Req rq = request_of(a, pool.page_shift, r);
    const int n_cols = (rq.row1 - rq.row0) * G;              // (token, head of the group) columns of this cache head
    const int span = sp.span(rq.len), used = sp.used(rq.len);
    if (n_cols <= 0 || (blockIdx.x && (int) blockIdx.x >= used)) {
        if (rest) wait_for_grid();
        return;
    }
    const int k0 = blockIdx.x * span, k1 = range_end(rq.len, k0, span);
    const int32_t * table = a.table + (size_t) r * a.width;
    const int n_pages = (int) (pool.n_slots >> pool.page_shift), pmask = (1 << pool.page_shift) - 1;
    uint8_t * ring = smem + warp * STAGES * SB;
    // addresses of this cache head: bytes from page to page and from keys to values, this lane's scales (lane = (plane,
    // group, quarter of a step), in the order in which a stage holds them) and its place among a copy's rows
    const uint32_t q_plane = ((uint32_t) pool.heads << pool.page_shift) * RB, q_page = 2 * q_plane;   // at most 2^25 bytes
    const uint8_t * q_head = pool.q + ((size_t) kh << pool.page_shift) * RB;
    const uint32_t d_page = ((uint32_t) 2 * pool.heads * NG) << pool.page_shift;
    const __half * d_lane = pool.d + ((((size_t) (lane / (4 * NG)) * pool.heads + kh) * NG + (lane / 4) % NG) << pool.page_shift) + 8 * (lane & 1);
    const uint32_t ring_s = smem_addr(ring);
    const uint32_t copy_dst = row_pos(lane / NG) * RB + 16 * chunk_pos<NG>(row_pos(lane / NG), lane % NG);
    // where this lane reads: its words of key row g, and of the value rows 2 t and 2 t + 1 (NG odd: half-words)
    const int k_at = row_pos(g) * RB + (NG == 4 ? 16 * chunk_pos<NG>(row_pos(g), t) : 4 * NG * t);
    const int v_a = row_pos(2 * t), v_b = row_pos(2 * t + 1);
    const int v_at[2] = {v_a * RB + (NG % 2 ? 2 * g : 16 * chunk_pos<NG>(v_a, g >> 2) + 4 * (g & 3)),
                         v_b * RB + (NG % 2 ? 2 * g : 16 * chunk_pos<NG>(v_b, g >> 2) + 4 * (g & 3))};
    // .. and from there to the second 64 channels (of four-chunk rows: the other two chunks, which side depends on the row)
    const int v_step[2] = {NG == 4 && (v_a & 2) ? -32 : 32, NG == 4 && (v_b & 2) ? -32 : 32};

    // rest: only the columns that the tiles kernel leaves
    for (int c0 = (rest ? tile_columns(n_cols) : 0) + (int) (blockIdx.y % tiles) * 8 * NT; c0 < n_cols; c0 += tiles * 8 * NT) {
        if (threadIdx.x < 8 * NT) s_poison[threadIdx.x] = 0;
        // ---- the tile's columns: lane (g, t) loads channels 32 i + 8 t .. + 7 of column g of each 8
        uint32_t qf[NT][NG][4];
        float sl2[NT][2];
        int lim[NT][2], low = 0x7fffffff;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int col = c0 + 8 * nt + g;
            const int row = rq.row0 + col / G, head = kh * G + col % G;
            if (threadIdx.x < 32 && t == 0) s_col[8 * nt + g] = make_int2(row, head);
            const T * q = (const T *) a.q + (long long) row * a.q_tok + head * a.q_head + 8 * t;
            float amax = 0.0f, x[NG][8];
#pragma unroll
            for (int i = 0; i < NG; i++) {
                T e[8];
                if (col >= n_cols) {
#pragma unroll
                    for (int c = 0; c < 8; c++) e[c] = to_type<T>(0.0f);
                } else if (vec & 1) {
                    *(uint4 *) e = *(const uint4 *) (q + 32 * i);
                } else {
#pragma unroll
                    for (int c = 0; c < 8; c++) e[c] = q[32 * i + c];
                }
#pragma unroll
                for (int c = 0; c < 8; c++) { x[i][c] = from_type(e[c]); amax = fmaxf(amax, fabsf(x[i][c])); }
            }
            int ex = 0;                                      // the row is multiplied by 2^ex
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            const int eb = (int) (__float_as_uint(amax) >> 23);        // biased exponent; 255: not finite
            if (amax > 0.0f && eb < 255) ex = min(14 - (eb - 127), 126);
            const float up = __int_as_float((127 + ex) << 23);
#pragma unroll
            for (int i = 0; i < NG; i++) {
#pragma unroll
                for (int c = 0; c < 4; c++) qf[nt][i][c] = pack_h2(x[i][c] * up, x[i][c + 4] * up);
            }
            // the factor of the scores of columns 2 t and 2 t + 1 (in log2 units), and the keys they see
            const float f = a.scale * 1.4426950408889634f * __int_as_float((127 - ex) << 23);
            const int see = col < n_cols ? visible(rq, row, a.frame) : 0x7fffffff;
#pragma unroll
            for (int e = 0; e < 2; e++) {
                sl2[nt][e] = __shfl_sync(0xffffffffu, f, 4 * (2 * t + e));
                lim[nt][e] = __shfl_sync(0xffffffffu, see, 4 * (2 * t + e));
                low = min(low, lim[nt][e]);
            }
        }
        low = min(low, __shfl_xor_sync(0xffffffffu, low, 1));
        low = min(low, __shfl_xor_sync(0xffffffffu, low, 2));

        // z: the running maximum less 10; weights are 2^(s - z). Before the first score: the lowest float, below which no
        // finite score lies
        float o[MT][NT][4], z[NT][2], l[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            z[nt][0] = z[nt][1] = -FLT_MAX;
            l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
            for (int i = 0; i < MT; i++) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.0f;
        }
        __syncthreads();                                     // s_poison is clear

        // ---- the ring: step i of this warp holds keys k0 + 32 (4 i + warp) ..; a step touches two pages at most
        const int steps = (max(0, k1 - k0) + STEP - 1) / STEP, mine = steps > warp ? (steps - warp + WARPS - 1) / WARPS : 0;
        auto page_at = [&](int key) -> int {
            const int i = key >> pool.page_shift;
            const int p = i < a.width && key < k1 ? __ldg(table + i) : -1;
            return p < n_pages ? p : -1;
        };
        int pg0 = -1, pg1 = -1;                              // the pages of the next step to be issued
        if (mine) { const int key = k0 + STEP * warp; pg0 = page_at(key); pg1 = page_at(key + 16); }
        uint32_t holes = 0;                                  // 2 bits a step, the oldest lowest: halves that have no page
        uint32_t fill = 0, read = 0;                         // byte offsets of the stage to be filled and read next
        auto issue = [&](int i) {
            if (i < mine) {
                // a half without a page copies page 0's rows, which are masked
                const int key = k0 + STEP * (WARPS * i + warp);
                const uint32_t dst = ring_s + fill;
                fill = fill == (STAGES - 1) * SB ? 0 : fill + SB;
                const uint8_t * src[2] = {q_head + (uint64_t) (uint32_t) max(pg0, 0) * q_page + (key & pmask) * RB,
                                          q_head + (uint64_t) (uint32_t) max(pg1, 0) * q_page + ((key + 16) & pmask) * RB};
#pragma unroll
                for (int e = 0; e < NG; e++) {               // 8 rows of 4 chunks (NG 4), 16 of 2, 32 of 1; NG 3: 32 chunks
                    const int c = lane + 32 * e, rr = c / NG, pos = row_pos(rr);
                    const uint8_t * x = NG == 3 ? (rr < 16 ? src[0] : src[1]) + (rr & 15) * RB + 16 * (c % NG)
                                     : NG == 1 ? (lane < 16 ? src[0] : src[1]) + (lane & 15) * 16
                                               : src[e * 32 / NG / 16] + lane * 16 + ((e * 32 / NG) & 15) * RB;
                    const uint32_t y = NG == 4 ? copy_dst + e * 8 * RB : NG == 2 ? copy_dst + e * 16 * RB
                                     : pos * RB + 16 * chunk_pos<NG>(pos, c % NG);
                    cp_async16(dst + y, x);
                    cp_async16(dst + y + STEP * RB, x + q_plane);
                }
                if (lane < 8 * NG) {                         // 8 scales at a time: (plane, group, quarter of the step)
                    const __half * x = (lane & 2 ? d_lane + (uint64_t) (uint32_t) max(pg1, 0) * d_page + ((key + 16) & pmask)
                                                 : d_lane + (uint64_t) (uint32_t) max(pg0, 0) * d_page + (key & pmask));
                    cp_async16(dst + 2 * STEP * RB + 16 * lane, x);
                }
                holes |= ((uint32_t) pg0 >> 31 | (uint32_t) pg1 >> 31 << 1) << (2 * (i < STAGES - 1 ? i : STAGES - 1));
                if (i + 1 < mine) { const int next = key + STEP * WARPS; pg0 = page_at(next); pg1 = page_at(next + 16); }
            }
            cp_async_commit();
        };
#pragma unroll
        for (int i = 0; i < STAGES - 1; i++) issue(i);

        for (int i = 0; i < mine; i++) {
            cp_async_wait<STAGES - 2>();
            __syncwarp();                                    // everyone's copies of step i are in, and step i - 1 is read
            issue(i + STAGES - 1);
            const uint32_t hole = holes & 3u;
            holes >>= 2;
            const uint8_t * kb = ring + read, * vb = kb + STEP * RB;
            read = read == (STAGES - 1) * SB ? 0 : read + SB;
            const __half * kd = (const __half *) (vb + STEP * RB), * vd = kd + NG * STEP;
            const int key = k0 + STEP * (WARPS * i + warp);
            // two tiles of 16 keys, one after the other (side by side in one body of twice the length: 142 us for 64 sessions of
            // 1000 .. 8190 keys instead of 120, and the counters showed stalls for instructions)
#pragma unroll 1
            for (int u = 0; u < 2; u++) {
                // ---- scores
                float s[NT][4];
                uint32_t w[2][NG];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint8_t * p = kb + k_at + (16 * u + 8 * h) * RB;
                    if (NG == 4) {
                        const uint4 x = *(const uint4 *) p;
                        w[h][0] = x.x; w[h][1 % NG] = x.y; w[h][2 % NG] = x.z; w[h][3 % NG] = x.w;
                    } else if (NG == 2) {
                        const uint2 x = *(const uint2 *) p;
                        w[h][0] = x.x; w[h][1 % NG] = x.y;
                    } else {
#pragma unroll
                        for (int gi = 0; gi < NG; gi++) w[h][gi] = *(const uint32_t *) (p + 4 * gi);
                    }
                }
#pragma unroll
                for (int gi = 0; gi < NG; gi++) {
                    __half2 x0[4], x1[4];
                    codes4(w[0][gi], x0);
                    codes4(w[1][gi], x1);
                    const float d0 = __half2float(kd[gi * STEP + 16 * u + g]), d1 = __half2float(kd[gi * STEP + 16 * u + 8 + g]);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        float acc[4];
                        mma16816_0(acc, {h2u(x0[0]), h2u(x1[0]), h2u(x0[1]), h2u(x1[1])}, qf[nt][gi][0], qf[nt][gi][1]);
                        mma16816(acc, {h2u(x0[2]), h2u(x1[2]), h2u(x0[3]), h2u(x1[3])}, qf[nt][gi][2], qf[nt][gi][3]);
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const float d = e < 2 ? d0 : d1;
                            s[nt][e] = gi == 0 ? d * acc[e] : __fmaf_rn(d, acc[e], s[nt][e]);
                        }
                    }
                }
                const bool whole = key + 16 * u + 16 <= min(low, k1) && !((hole >> u) & 1);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                    for (int e = 0; e < 4; e++) s[nt][e] *= sl2[nt][e & 1];
                }
                if (!whole) {
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int k = key + 16 * u + 8 * (e >> 1) + g;
                            if (k >= min(lim[nt][e & 1], k1) || ((hole >> u) & 1)) s[nt][e] = -INFINITY;
                        }
                    }
                    asm volatile("" ::: "memory");               // keeps the masks out of the steps that need none
                }
                float mx[NT][2];
                bool raise = false;
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        mx[nt][e] = fmaxf(s[nt][e], s[nt][e + 2]);
                        raise = raise || mx[nt][e] - z[nt][e] > 14.0f;
                    }
                }
                if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            float x = mx[nt][e];
#pragma unroll
                            for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                            x = fmaxf(below(x), z[nt][e]);
                            const float c = x == z[nt][e] ? 1.0f : ex2(z[nt][e] - x);
                            z[nt][e] = x;
                            l[nt][e] *= c;
#pragma unroll
                            for (int k = 0; k < MT; k++) { o[k][nt][e] *= c; o[k][nt][e + 2] *= c; }
                        }
                    }
                }
                // ---- weights, as the B operand of the second product
                uint32_t pf[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    const float p0 = ex2(s[nt][0] - z[nt][0]), p1 = ex2(s[nt][1] - z[nt][1]);
                    const float p2 = ex2(s[nt][2] - z[nt][0]), p3 = ex2(s[nt][3] - z[nt][1]);
                    l[nt][0] += p0 + p2;
                    l[nt][1] += p1 + p3;
                    pf[nt][0] = transpose8(pack_h2(p0, p1));
                    pf[nt][1] = transpose8(pack_h2(p2, p3));
                }
            // ---- sums of values
                const int ra = 16 * u + 2 * t;                         // this lane's keys: ra, ra + 1, ra + 8, ra + 9
                constexpr int PARTS = NG % 2 ? NG : NG / 2;           // 32 or 64 channels at a time
#pragma unroll
                for (int j = 0; j < PARTS; j++) {
                    const int grp = NG % 2 ? j : 2 * j + (g >> 2);
                    __half2 d0 = *(const __half2 *) (vd + grp * STEP + ra), d1 = *(const __half2 *) (vd + grp * STEP + ra + 8);
                    if (!whole) {
                        // a weight of 0 does not silence a value that is not a number: such scales become 0 here, and the
                        // columns that see the key get their NaN at the end
                        const __half e[4] = {__low2half(d0), __high2half(d0), __low2half(d1), __high2half(d1)};
                        __half f[4];
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            f[c] = e[c];
                            if (__hisnan(e[c]) || __hisinf(e[c])) {
                                f[c] = __ushort_as_half(0);
                                const int k = key + ra + (c & 1) + 8 * (c >> 1);
                                for (int col = 0; col < 8 * NT && !((hole >> u) & 1); col++) {
                                    const int cc = c0 + col;
                                    if (cc < n_cols && k < k1 && k < visible(rq, s_col[col].x, a.frame)) atomicOr(&s_poison[col], 1u << grp);
                                }
                            }
                        }
                        d0 = __halves2half2(f[0], f[1]);
                        d1 = __halves2half2(f[2], f[3]);
                    }
                    uint32_t w[4];
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        const uint8_t * p = vb + v_at[c & 1] + (16 * u + 8 * (c >> 1)) * RB;
                        if (NG % 2) w[c] = *(const uint16_t *) (p + 16 * j);
                        else w[c] = *(const uint32_t *) (j ? p + v_step[c & 1] : p);
                    }
#pragma unroll
                    for (int h = 0; h < (NG % 2 ? 1 : 2); h++) {
                        const uint32_t sel = h ? 0x7632 : 0x5410;      // half h of one key's word beside the next key's
                        __half2 x[4], y[4];
                        codes4(__byte_perm(w[0], w[1], sel), x);
                        codes4(__byte_perm(w[2], w[3], sel), y);
#pragma unroll
                        for (int c = 0; c < 4; c++) { x[c] = __hmul2(x[c], d0); y[c] = __hmul2(y[c], d1); }
                        const int mt = NG % 2 ? 2 * j : 4 * j + 2 * h;
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            mma16816(o[mt][nt], {h2u(x[0]), h2u(x[1]), h2u(y[0]), h2u(y[1])}, pf[nt][0], pf[nt][1]);
                            mma16816(o[mt + 1][nt], {h2u(x[2]), h2u(x[3]), h2u(y[2]), h2u(y[3])}, pf[nt][0], pf[nt][1]);
                        }
                    }
                }
            }
        }
        cp_async_wait<0>();
        __syncthreads();                                     // the rings become the merge's buffers

        // ---- merge the four warps: [warp][column][hd + 4], then (maximum, sum) [warp][column]
        float * so = (float *) smem;
        float2 * sm = (float2 *) (so + WARPS * 8 * NT * (HD + 4));
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int e = 0; e < 2; e++) {
                float x = l[nt][e];
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
                const int col = warp * 8 * NT + 8 * nt + 2 * t + e;
                if (g == 0) sm[col] = make_float2(z[nt][e], x);
#pragma unroll
                for (int k = 0; k < MT; k++) {
                    const int c = NG % 2 ? 32 * (k / 2) + 4 * g + 2 * (k % 2) : 64 * (k / 4) + 8 * g + 2 * (k % 4);
                    *(float2 *) (so + col * (HD + 4) + c) = make_float2(o[k][nt][e], o[k][nt][e + 2]);
                }
            }
        }
        __syncthreads();
        for (int idx = threadIdx.x; idx < 8 * NT * (HD / 4); idx += 32 * WARPS) {
            const int col = idx / (HD / 4), c = idx % (HD / 4) * 4;
            if (c0 + col >= n_cols) continue;
            float top = -FLT_MAX, sum = 0.0f;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < WARPS; w++) top = fmaxf(top, sm[w * 8 * NT + col].x);
#pragma unroll
            for (int w = 0; w < WARPS; w++) {
                // (a warp that saw nothing has zeros, or what a score that is not a number has made of them: kept by 0 * NaN)
                const float2 ml = sm[w * 8 * NT + col];
                const float f = ml.x == top ? 1.0f : ex2(ml.x - top);
                const float4 x = *(const float4 *) (so + (w * 8 * NT + col) * (HD + 4) + c);
                sum = __fmaf_rn(ml.y, f, sum);
                v.x = __fmaf_rn(x.x, f, v.x); v.y = __fmaf_rn(x.y, f, v.y); v.z = __fmaf_rn(x.z, f, v.z); v.w = __fmaf_rn(x.w, f, v.w);
            }
            if ((s_poison[col] >> (c / 32)) & 1) v.x = v.y = v.z = v.w = __int_as_float(0x7fffffff);
            const int row = s_col[col].x, head = s_col[col].y;
            if (used <= 1) {
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                T * out = (T *) a.out + (long long) row * a.o_tok + head * a.o_head + c;
                const T y[4] = {to_type<T>(v.x * inv), to_type<T>(v.y * inv), to_type<T>(v.z * inv), to_type<T>(v.w * inv)};
                if (vec & 2) {
                    uint2 w;
                    memcpy(&w, y, 8);
                    *(uint2 *) out = w;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) out[e] = y[e];
                }
            } else {
                const size_t at = ((size_t) blockIdx.x * a.n_rows + row) * a.heads + head;
                *(float4 *) (sp.o + at * HD + c) = v;
                if (c == 0) sp.ml[at] = make_float2(top, sum);
            }
        }
        __syncthreads();
    }
    if (rest) wait_for_grid();
}

// Joins the partial sums of a row: one CTA per (row, head), its warps taking every eighth part.
template <class T, int NG>
__global__ void __launch_bounds__(256) k_kv4_merge(const Kv4Pool pool, const Kv4Attn a, const Split sp) {
    constexpr int HD = 32 * NG;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __shared__ float s_top[8], s_sum[8], s_o[8][HD];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, head = blockIdx.y;
    const Req rq = request_of(a, pool.page_shift, blockIdx.z);
    const int used = sp.used(rq.len);
    if (used <= 1) return;                                   // written by the first kernel
    for (int row = rq.row0 + blockIdx.x; row < rq.row1; row += gridDim.x) {
        const size_t at = (size_t) row * a.heads + head, step = (size_t) a.n_rows * a.heads;
        float top = -FLT_MAX;
        for (int s = threadIdx.x; s < used; s += 256) top = fmaxf(top, sp.ml[at + s * step].x);
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        if (lane == 0) s_top[warp] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 8; w++) top = fmaxf(top, s_top[w]);
        float sum = 0.0f, v[NG];
#pragma unroll
        for (int i = 0; i < NG; i++) v[i] = 0.0f;
#pragma unroll 4
        for (int s = warp; s < used; s += 8) {
            const float2 ml = sp.ml[at + s * step];
            const float f = ml.x == top ? 1.0f : ex2(ml.x - top);
            sum = __fmaf_rn(ml.y, f, sum);
#pragma unroll
            for (int i = 0; i < NG; i++) v[i] = __fmaf_rn(sp.o[(at + s * step) * HD + 32 * i + lane], f, v[i]);
        }
#pragma unroll
        for (int i = 0; i < NG; i++) s_o[warp][32 * i + lane] = v[i];
        if (lane == 0) s_sum[warp] = sum;
        __syncthreads();
        for (int c = threadIdx.x; c < HD; c += 256) {
            float x = 0.0f, z = 0.0f;
#pragma unroll
            for (int w = 0; w < 8; w++) { x += s_o[w][c]; z += s_sum[w]; }
            ((T *) a.out)[(long long) row * a.o_tok + head * a.o_head + c] = to_type<T>(z == 0.0f ? x * 0.0f : x / z);
        }
        __syncthreads();
    }
}

// The launch: which kernel, columns a CTA takes, CTAs along the columns, and the division of the keys. Counts of the whole
// grid are taken in 64 bits: n_req, heads * tiles and max_len have 16, 16 and 31, and their product 63.
struct Plan {
    bool tc;                    // the tiles kernel
    int nt, tiles;
    Split sp;
};
Plan plan_of(const Kv4Pool & p, const Kv4Attn & a) {
    Plan r;
    const long long group = a.heads / p.heads, cols = a.max_new * group;
    r.tc = cols > FEW;
    r.nt = (r.tc ? cols % 256 : cols) > 8 ? 2 : 1;
    if (r.tc) r.tiles = (int) std::min<long long>((cols + 255 - FEW) / 256, 65535 / p.heads);
    else r.tiles = (int) std::min<long long>((cols + 8 * r.nt - 1) / (8 * r.nt), 65535 / p.heads);
    // CTAs along requests and columns; where the rows of a request are not known, all requests together have n_rows
    long long ctas = (long long) a.n_req * r.tiles;
    if (a.max_new >= a.n_rows) ctas = std::min(ctas, a.n_req + a.n_rows * group / (r.tc ? 256 : 8 * r.nt));
    // Ranges of 1024 keys or more, 4 to each of the 148 SMs x 4 resident CTAs if every request is as long as the longest
    // (fewer leave SMs idle at the end where lengths differ, more pay for starts and partial sums; 64 sessions of
    // 1000 .. 8190 keys: 768 / 1536 / 2048 / 4096 keys a range = 121 / 115 / 116 / 126 us); down to 256 keys when a range
    // for each CTA is shorter than that.
    const long long total = ctas * p.heads * a.max_len, slots = r.tc ? 148 : 148 * 4;
    const long long whole = (a.max_len + 127LL) & ~127LL;
    long long chunk = (std::max(std::max(256LL, std::min(1024LL, total / slots)), total / (4 * slots)) + 127) & ~127LL;
    // One range where a second would be short or small: it would cost a second kernel, and for many rows their partial sums.
    // One range against ranges of 256 keys, us, replayed one after the other: one row of 16 heads of 64, 300 / 516 / 768 keys,
    // 1 session 5.5 / 7.1 / 7.6 and 7.0 / 7.2 / 7.2, 32 sessions 8.1 / 11.9 / 14.2 and 8.1 / 25.4 / 14.2; 8 cache heads of
    // 128, 1 session 7.4 / 9.9 / 10.5 and 8.6 / 8.6 / 8.6, 32 sessions 9.2 / 13.8 / 15.5 and 24.0 / 31.7 / 28.7; 128 rows of 16
    // heads of 64, 1 session 11.8 / 15.2 / 17.9 and 32.8 / 32.9 / 33.0. So at most 2 us are lost, where a single session has
    // few cache heads and 500 keys and more. (Behind 768 keys many rows of few sessions pay for it: those 128 rows take
    // 33 us at 800 keys, of 4 sessions 100 us instead of 18 at 768.)
    if (a.max_len <= 768 || a.max_len <= chunk + chunk / 4) chunk = whole;
    r.sp.chunk = (int) chunk;                                // at most `whole`, which is below 2^31 (attn_of)
    r.sp.n_split = (int) ((a.max_len + chunk - 1) / chunk);
    r.sp.o = nullptr;
    r.sp.ml = nullptr;
    return r;
}

size_t partial_bytes(const Kv4Pool & p, const Kv4Attn & a, int n_split) {
    return n_split <= 1 ? 0 : (size_t) n_split * a.n_rows * a.heads * (p.hd + 2) * 4;
}

template <class T, int NG, int NT>
int rows_launch(const Kv4Pool & p, const Kv4Attn & a, const Plan & r, int vec, cudaStream_t st) {
    const int tiles = !r.tc ? r.tiles : NT == 1 ? 1 : 2;      // beside the tiles kernel: the columns it leaves
    constexpr int smem = rows_smem<NG, NT>();
    if (allow_smem<k_kv4_rows<T, NG, NT>>(smem)) return -1;
    const dim3 grid((unsigned) r.sp.n_split, (unsigned) (p.heads * tiles), (unsigned) a.n_req);
    JB_CUDA(launch_pdl(k_kv4_rows<T, NG, NT>, grid, dim3(32 * WARPS), smem, st, p, a, r.sp, tiles, vec, r.tc ? 1 : 0));
    return 0;
}

template <class T, int NG>
int launch(const Kv4Pool & p, const Kv4Attn & a, const Kv4Waits & waits, cudaStream_t st) {
    Plan r = plan_of(p, a);
    if (r.sp.n_split > 1) {
        r.sp.o = (float *) a.ws;
        r.sp.ml = (float2 *) (r.sp.o + (size_t) r.sp.n_split * a.n_rows * a.heads * p.hd);
    }
    // 16-byte loads of q, 8- and 16-byte stores of out where the strides allow them
    const int vec = (((uintptr_t) a.q & 15) == 0 && ((a.q_tok | a.q_head) & 7) == 0 ? 1 : 0) |
                    (((uintptr_t) a.out & 7) == 0 && ((a.o_tok | a.o_head) & 3) == 0 ? 2 : 0) |
                    (((uintptr_t) a.out & 15) == 0 && ((a.o_tok | a.o_head) & 7) == 0 ? 4 : 0);
    if (r.tc && kv4_tiles(p, a, waits, r.sp, r.tiles, vec, st)) return -1;
    if (r.nt == 1 ? rows_launch<T, NG, 1>(p, a, r, vec, st) : rows_launch<T, NG, 2>(p, a, r, vec, st)) return -1;
    if (r.sp.n_split > 1) {
        // (a CTA walks rows of its request from its own on: max_new may be unknown, and then far too many)
        const dim3 grid((unsigned) std::min(std::max(1, a.max_new), 64), (unsigned) a.heads, (unsigned) a.n_req);
        JB_CUDA(launch_pdl(k_kv4_merge<T, NG>, grid, dim3(256), 0, st, p, a, r.sp));
    }
    return 0;
}

template <class T>
int launch_dim(const Kv4Pool & p, const Kv4Attn & a, const Kv4Waits & waits, cudaStream_t st) {
    switch (p.hd / 32) {
        case 1: return launch<T, 1>(p, a, waits, st);
        case 2: return launch<T, 2>(p, a, waits, st);
        case 3: return launch<T, 3>(p, a, waits, st);
        default: return launch<T, 4>(p, a, waits, st);
    }
}

}  // namespace

size_t kv4_attention_workspace(const Kv4Pool & p, const Kv4Attn & a) {
    if (!a.n_req || !a.n_rows) return 0;
    return partial_bytes(p, a, plan_of(p, a).sp.n_split);
}

void kv4_attention_plan(const Kv4Pool & p, const Kv4Attn & a, int * out) {
    const Plan r = plan_of(p, a);
    out[0] = r.tc;
    out[1] = r.tiles;
    out[2] = r.sp.n_split;
    out[3] = r.sp.chunk;
}

int kv4_attention(const Kv4Pool & p, const Kv4Attn & a, const Kv4Waits & w, cudaStream_t st) {
    KTimer kt("kv4_attention", st);
    return a.type == KV4_F16 ? launch_dim<__half>(p, a, w, st) : launch_dim<__nv_bfloat16>(p, a, w, st);
}

}  // namespace jb
