// Attention over the paged 4-bit cache (kv4.h).
//
//   row i of request r (of n = q_start[r + 1] - q_start[r]) stands at position p = lens[r] - n + i and sees the keys
//   j < lens[r], and with frame > 0 only j < (p / frame + 1) frame (none for p < 0):
//   out = sum_j w_j v_j / sum_j w_j,  w_j = exp(scale q . k_j - max);  0 for a row that sees nothing.
#include "kv4.h"
#include "common.h"
#include "launch.h"
#include "kprof.h"

#include <cuda_bf16.h>

namespace jb {

namespace {

__device__ __forceinline__ float from_type(__half x) { return __half2float(x); }
__device__ __forceinline__ float from_type(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T> __device__ __forceinline__ T to_type(float x);
template <> __device__ __forceinline__ __half to_type(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 to_type(float x) { return __float2bfloat16_rn(x); }

// keys row p (its position) sees
__device__ __forceinline__ int visible(int p, int len, int frame) {
    if (frame == 0) return len;
    if (p < 0) return 0;
    const long long lim = ((long long) p / frame + 1) * frame;
    return lim < len ? (int) lim : len;
}

// one warp per (row, head), lane c holding channels c, c + 32, ..
template <class T, int NG>
__global__ void __launch_bounds__(128) k_kv4_attention(const Kv4Pool pool, const Kv4Attn a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int h = blockIdx.y, r = blockIdx.z, kh = h / (a.heads / pool.heads);
    const int q0 = max(0, a.q_start[r]), n = min(a.q_start[r + 1], a.n_rows) - q0;
    const int P = 1 << pool.page_shift;
    const int len = (int) min((long long) max(a.lens[r], 0), (long long) a.width << pool.page_shift);
    const long long pages = pool.n_slots >> pool.page_shift;
    for (int i = blockIdx.x * 4 + warp; i < n; i += gridDim.x * 4) {
        const int keys = visible(a.lens[r] - n + i, len, a.frame);
        float q[NG], acc[NG];
#pragma unroll
        for (int g = 0; g < NG; g++) {
            q[g] = from_type(((const T *) a.q)[(long long) (q0 + i) * a.q_tok + h * a.q_head + 32 * g + lane]);
            acc[g] = 0.0f;
        }
        float m = -INFINITY, l = 0.0f;
        for (int j = 0; j < keys; j++) {
            const int page = a.table[(size_t) r * a.width + (j >> pool.page_shift)];
            if (page < 0 || page >= pages) continue;
            const int row = j & (P - 1);
            const uint8_t * kq = pool.q + kv4_q_at(pool, page, 0, kh, row), * vq = pool.q + kv4_q_at(pool, page, 1, kh, row);
            const __half * kd = pool.d + kv4_d_at(pool, page, 0, kh, row), * vd = pool.d + kv4_d_at(pool, page, 1, kh, row);
            float s = 0.0f;
#pragma unroll
            for (int g = 0; g < NG; g++) {
                const uint32_t b = kq[((lane >> 3) * NG + g) * 4 + ((lane & 7) >> 1)];
                s += q[g] * ((float) ((int) ((b >> (4 * (lane & 1))) & 15u) - 8) * __half2float(kd[(size_t) g * P]));
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            s *= a.scale;
            const float nm = fmaxf(m, s), c = m == nm ? 1.0f : expf(m - nm), w = s == nm ? 1.0f : expf(s - nm);
            m = nm;
            l = l * c + w;
#pragma unroll
            for (int g = 0; g < NG; g++) {
                const uint32_t b = vq[16 * g + (lane >> 1)];
                acc[g] = acc[g] * c + w * ((float) ((int) ((b >> (4 * (lane & 1))) & 15u) - 8) * __half2float(vd[(size_t) g * P]));
            }
        }
        const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
#pragma unroll
        for (int g = 0; g < NG; g++) {
            ((T *) a.out)[(long long) (q0 + i) * a.o_tok + h * a.o_head + 32 * g + lane] = to_type<T>(acc[g] * inv);
        }
    }
}

template <class T>
int launch(const Kv4Pool & p, const Kv4Attn & a, cudaStream_t st) {
    const dim3 grid((unsigned) ((a.max_new + 3) / 4), (unsigned) a.heads, (unsigned) a.n_req);
    switch (p.hd / 32) {
        case 1: JB_CUDA(launch_pdl(k_kv4_attention<T, 1>, grid, dim3(128), 0, st, p, a)); break;
        case 2: JB_CUDA(launch_pdl(k_kv4_attention<T, 2>, grid, dim3(128), 0, st, p, a)); break;
        case 3: JB_CUDA(launch_pdl(k_kv4_attention<T, 3>, grid, dim3(128), 0, st, p, a)); break;
        default: JB_CUDA(launch_pdl(k_kv4_attention<T, 4>, grid, dim3(128), 0, st, p, a)); break;
    }
    return 0;
}

}  // namespace

size_t kv4_attention_workspace(const Kv4Pool &, const Kv4Attn &) { return 0; }

int kv4_attention(const Kv4Pool & p, const Kv4Attn & a, cudaStream_t st) {
    KTimer kt("kv4_attention", st);
    return a.type == KV4_F16 ? launch<__half>(p, a, st) : launch<__nv_bfloat16>(p, a, st);
}

}  // namespace jb
