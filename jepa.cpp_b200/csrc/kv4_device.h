// Device-side pieces that the two kernels of kv4_attention share: a request's rows and keys, the division of the
// keys over CTAs, and the conversion of 4-bit codes.
#pragma once

#include "kv4.h"
#include "common.h"

#include <cuda_bf16.h>

#include <atomic>

namespace jb {

template <class T> __device__ __forceinline__ T to_type(float x);
template <> __device__ __forceinline__ __half to_type(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 to_type(float x) { return __float2bfloat16_rn(x); }
__device__ __forceinline__ float from_type(__half x) { return __half2float(x); }
__device__ __forceinline__ float from_type(__nv_bfloat16 x) { return __bfloat162float(x); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// how a request's keys are divided: n_split ranges of `chunk` keys, longer ones where that does not cover them
struct Split {
    int n_split, chunk;
    float * o;                  // [n_split][n_rows][heads][hd] partial sums
    float2 * ml;                // [n_split][n_rows][heads] (maximum, sum)
    __host__ __device__ int span(int len) const {
        const int even = (int) (((long long) len + n_split - 1) / n_split);
        return even <= chunk ? chunk : (even + 127) & ~127;
    }
    __host__ __device__ int used(int len) const { return len > 0 ? (len - 1) / span(len) + 1 : 0; }
};

// end of the range of `span` keys that starts at k0 (k0 + span may pass 2^31)
__device__ __forceinline__ int range_end(int len, int k0, int span) { return len - k0 < span ? len : k0 + span; }

// What a CTA needs to know of its request: rows [row0, row1) of q, keys [0, len) of the table. Whatever q_start holds,
// 0 <= row0 <= row1 <= n_rows, so that row1 - row0 cannot overflow into a count of rows; a row that is there has last > row.
struct Req {
    int row0, row1, last, len;
};
__device__ __forceinline__ Req request_of(const Kv4Attn & a, int page_shift, int r) {
    Req q;
    q.last = a.q_start[r + 1];
    q.row0 = min(max(0, a.q_start[r]), a.n_rows);
    q.row1 = max(q.row0, min(q.last, a.n_rows));
    q.len = (int) min((long long) max(a.lens[r], 0), (long long) a.width << page_shift);
    return q;
}
// keys that row `row` sees
__device__ __forceinline__ int visible(const Req & q, int row, int frame) {
    if (frame == 0) return q.len;
    const int p = q.len - q.last + row;
    if (p < 0) return 0;
    const long long lim = ((long long) p / frame + 1) * frame;
    return lim < q.len ? (int) lim : q.len;
}

// Columns of a request and cache head that the tiles kernel takes, of n in all: whole tiles of 256, and what is left over if
// it is more than 32; the rows kernel takes the rest, 16 at a time. 32 sessions of 6000 .. 8000 keys, 4 cache heads, head_dim 64 / 128:
// 24 columns take the rows kernel 90 / 137 us and the tiles kernel 135 / 197, 32 columns 101 / 150 and 141 / 204; a third
// and fourth pass over the cache would cost more than the tiles kernel there: 40 / 48 / 64 columns of 32 sessions of 7000 keys,
// 16 heads of 64, 579 / 631 / 403 us against 387. (258 columns in two CTAs of the tiles kernel: the second, for 2 of
// them, took as long as the first.) The border costs something on either side: 32 columns of those 32 sessions of 16 heads
// take 442 us and would take 387 as tiles; 40 and 48 columns of 1 to 8 sessions would mostly be 5 to 40 % faster in the rows
// kernel (one session of 500 keys, 16 heads of 64: 7.8 us against 13.6; 4000 keys, 8 heads of 128: 17.9 against 21.0).
constexpr int FEW = 32;
__host__ __device__ inline int tile_columns(int n) { return n % 256 > FEW ? n : n - n % 256; }

__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *(const uint32_t *) &h;
}
__device__ __forceinline__ uint32_t h2u(__half2 h) { return *(const uint32_t *) &h; }
__device__ __forceinline__ __half2 u2h(uint32_t u) { return *(const __half2 *) &u; }

// The nibbles 0 .. 3 of both 16-bit halves of u as four half2 of the integers -8 .. 7: 0x6400 | c is 1024 + c in f16,
// 0x6400 | 16 c is 1024 + 16 c; both steps are exact.
__device__ __forceinline__ uint32_t and_or(uint32_t u, uint32_t mask) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(u), "r"(mask), "r"(0x64006400u));
    return r;
}
__device__ __forceinline__ void codes4(uint32_t u, __half2 (&x)[4]) {
    const __half2 bias = u2h(0xe408e408u), sixteenth = u2h(0x2c002c00u), bias16 = u2h(0xd480d480u);   // -1032, 1/16, -72
    const uint32_t v = u >> 8;
    x[0] = __hadd2(u2h(and_or(u, 0x000f000fu)), bias);
    x[1] = __hfma2(u2h(and_or(u, 0x00f000f0u)), sixteenth, bias16);
    x[2] = __hadd2(u2h(and_or(v, 0x000f000fu)), bias);
    x[3] = __hfma2(u2h(and_or(v, 0x00f000f0u)), sixteenth, bias16);
}

// Lets kernel K have `bytes` of dynamic shared memory, once a device.
template <auto K>
int allow_smem(int bytes) {
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    JB_CUDA(cudaGetDevice(&dev));
    const uint64_t bit = (uint64_t) 1 << (dev & 63);
    if (dev < 64 && (done.load(std::memory_order_relaxed) & bit)) return 0;
    JB_CUDA(cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    if (dev < 64) done.fetch_or(bit, std::memory_order_relaxed);
    return 0;
}

// The tiles kernel (kv4_attention_tc.cu): `grid` = (key ranges, cache heads x tiles of 256 columns, requests).
int kv4_tiles(const Kv4Pool & p, const Kv4Attn & a, const Kv4Waits & waits, const Split & sp, int tiles, int vec, cudaStream_t st);

}  // namespace jb
