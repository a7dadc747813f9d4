// Store and load of the 4-bit key / value cache, and the block tables and slot maps of a step (kv4.h).
#include "kv4.h"
#include "common.h"
#include "launch.h"
#include "kprof.h"

#include <cuda_bf16.h>

#include <algorithm>

namespace jb {

namespace {

// ------------------------------------------------------------------------------------------
// Store and load. A warp takes 8 tokens of one head, 4 lanes a token; lane t of a token holds channels
// 32 g + 8 t .. + 7 of every group g. So the 4 lanes of a token agree on a group's scale with two shuffles, a
// lane's key words lie side by side in the row, and the 8 tokens' scales of a group are 8 neighbours in memory
// (when the tokens are neighbours in a page, as the rows of a sequence are).
// ------------------------------------------------------------------------------------------

template <class T> struct Vec8;
template <> struct Vec8<__half> { uint4 a; };
template <> struct Vec8<__nv_bfloat16> { uint4 a; };
template <> struct Vec8<float> { uint4 a, b; };

// 8 elements from p; vec: p is 16-byte aligned
template <class T>
__device__ __forceinline__ Vec8<T> load8(const T * p, bool vec) {
    Vec8<T> v;
    if (vec) {
        v = *(const Vec8<T> *) p;
    } else {
        T e[8];
#pragma unroll
        for (int i = 0; i < 8; i++) e[i] = p[i];
        memcpy(&v, e, sizeof(v));
    }
    return v;
}

template <class T>
__device__ __forceinline__ void unpack8(const Vec8<T> & v, float (&x)[8]);
template <> __device__ __forceinline__ void unpack8(const Vec8<float> & v, float (&x)[8]) { memcpy(x, &v, 32); }
template <> __device__ __forceinline__ void unpack8(const Vec8<__half> & v, float (&x)[8]) {
    const __half2 * h = (const __half2 *) &v;
#pragma unroll
    for (int i = 0; i < 4; i++) { const float2 f = __half22float2(h[i]); x[2 * i] = f.x; x[2 * i + 1] = f.y; }
}
template <> __device__ __forceinline__ void unpack8(const Vec8<__nv_bfloat16> & v, float (&x)[8]) {
    const __nv_bfloat162 * h = (const __nv_bfloat162 *) &v;
#pragma unroll
    for (int i = 0; i < 4; i++) { const float2 f = __bfloat1622float2(h[i]); x[2 * i] = f.x; x[2 * i + 1] = f.y; }
}

// maximum and minimum that keep a NaN
__device__ __forceinline__ float max_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float min_nan(float a, float b) { float r; asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }

// The scale of a group whose largest and smallest values are hi and lo: the value of largest magnitude (the positive
// one of two) over -8, so that it takes code 0 and the 16 codes are used in full; rounded to bf16 (8 significant bits,
// see kv4.h), then to f16, which the clamp keeps in range (8160 * 8 < 65504). A group with an infinity or a NaN gets NaN.
__device__ __forceinline__ __half group_scale(float hi, float lo) {
    const float m = hi >= -lo ? hi : lo;
    const float r = __bfloat162float(__float2bfloat16_rn(m * -0.125f));
    const float d = fminf(fmaxf(r, -8160.0f), 8160.0f);
    const bool finite = hi - hi == 0.0f && lo - lo == 0.0f;   // false for infinities and NaN
    return finite ? __float2half_rn(d) : __ushort_as_half((unsigned short) 0x7fff);
}

// 2^23 + code in the bits of a float, code = clamp(floor(x / d + 1/2) + 8, 0, 15); inv is 1 / d within 2^-23 of itself.
// For f16 and bf16 x the quotient of an 11-bit by an 8-bit significand is a half-integer or at least 2^-13 away
// from one (for |quotient| between 1/2 and 8.1), and x * inv is within 2^-19 of it: adding 2^-15 decides every case as the
// exact quotient would. The clamp is the saturation of (quotient + 8.5) / 16 to [0, 1], and the factor a step below 16
// sends 1 to 15 (it moves the rest by 2^-20 at most). For f32 x the estimate is corrected by the sign of
// x - (c -+ 1/2) d, one fused rounding each.
template <class T>
__device__ __forceinline__ uint32_t code_of(float x, float d, float inv16) {
    const float t = __saturatef(__fmaf_rn(x, inv16, (8.5f + 0x1p-15f) * 0.0625f));
    uint32_t u = __float_as_uint(__fmaf_rd(t, 15.999999f, 8388608.0f));
    if (sizeof(T) == 4) {
        const uint32_t c = u & 15u;
        const float s = d < 0.0f ? -1.0f : 1.0f;
        const float k = (float) c - 8.0f;
        const float below = __fmaf_rn(-(k - 0.5f), d, x) * s, above = __fmaf_rn(-(k + 0.5f), d, x) * s;
        if (below < 0.0f && c > 0) u--;
        else if (above >= 0.0f && c < 15) u++;
    }
    return u;
}

template <class T, int NG>
__device__ __forceinline__ void quantise_row(const Vec8<T> (&in)[NG], uint32_t (&word)[NG], __half (&scale)[NG]) {
#pragma unroll
    for (int g = 0; g < NG; g++) {
        float x[8];
        unpack8<T>(in[g], x);
        float hi = x[0], lo = x[0];
#pragma unroll
        for (int i = 1; i < 8; i++) { hi = max_nan(hi, x[i]); lo = min_nan(lo, x[i]); }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
            lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        }
        scale[g] = group_scale(hi, lo);
        const float d = __half2float(scale[g]);
        const bool zero = d == 0.0f || d != d;
        float inv;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(zero ? 1.0f : d));
        inv *= 0.0625f;
        // the codes' words add up with weights 16^i; the 2^23 that each carries adds up to 0xfb000000 modulo 2^32
        uint32_t w = 0;
#pragma unroll
        for (int i = 7; i >= 0; i--) w = w * 16u + code_of<T>(x[i], d, inv);
        word[g] = zero ? 0x88888888u : w - 0xfb000000u;
    }
}

template <class T, int NG>
__global__ void __launch_bounds__(128) k_kv4_store(const Kv4Pool p, const Kv4Rows r, const int64_t * __restrict__ slots, long long n,
                                                   bool vec) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int lane = threadIdx.x & 31, t = lane & 3;
    const long long task = (long long) blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int h = (int) (task % p.heads);
    const long long tok = (task / p.heads) * 8 + (lane >> 2);
    if (task / p.heads * 8 >= n) return;                       // the whole warp
    const long long slot = tok < n ? slots[tok] : -1;
    const bool live = slot >= 0 && slot < p.n_slots;
    const long long row = live ? tok : task / p.heads * 8;     // a row that exists, for the shuffles' sake
    const T * k = (const T *) r.k + row * r.k_tok + h * r.k_head + 8 * t;
    const T * v = (const T *) r.v + row * r.v_tok + h * r.v_head + 8 * t;
    Vec8<T> kin[NG], vin[NG];
#pragma unroll
    for (int g = 0; g < NG; g++) kin[g] = load8<T>(k + 32 * g, vec);
#pragma unroll
    for (int g = 0; g < NG; g++) vin[g] = load8<T>(v + 32 * g, vec);
    uint32_t kw[NG], vw[NG];
    __half ks[NG], vs[NG];
    quantise_row<T, NG>(kin, kw, ks);
    quantise_row<T, NG>(vin, vw, vs);
    if (!live) return;
    const long long page = slot >> p.page_shift;
    const int at = (int) (slot & ((1 << p.page_shift) - 1)), P = 1 << p.page_shift;
    uint32_t * kq = (uint32_t *) (p.q + kv4_q_at(p, page, 0, h, at)) + t * NG;
    if (NG == 4) *(uint4 *) kq = make_uint4(kw[0], kw[1 % NG], kw[2 % NG], kw[3 % NG]);
    else if (NG == 2) *(uint2 *) kq = make_uint2(kw[0], kw[1 % NG]);
    else {
#pragma unroll
        for (int g = 0; g < NG; g++) kq[g] = kw[g];
    }
    uint32_t * vq = (uint32_t *) (p.q + kv4_q_at(p, page, 1, h, at));
#pragma unroll
    for (int g = 0; g < NG; g++) vq[4 * g + t] = vw[g];
    __half * kd = p.d + kv4_d_at(p, page, 0, h, at);
    __half * vd = p.d + kv4_d_at(p, page, 1, h, at);
#pragma unroll
    for (int g = 0; g < NG; g++) {
        if (t == g) { kd[(size_t) g * P] = ks[g]; vd[(size_t) g * P] = vs[g]; }
    }
}

template <class T> __device__ __forceinline__ T to_type(float x);
template <> __device__ __forceinline__ float to_type(float x) { return x; }
template <> __device__ __forceinline__ __half to_type(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 to_type(float x) { return __float2bfloat16_rn(x); }

// values d (c - 8) of N codes, rounded once to T (f16 and f32 hold them exactly): 16 bytes
template <class T, int N>
__device__ __forceinline__ void write16(T * p, uint32_t w, float d, bool live) {
    T e[N];
#pragma unroll
    for (int i = 0; i < N; i++) e[i] = to_type<T>(live ? (float) ((int) ((w >> (4 * i)) & 15u) - 8) * d : 0.0f);
    uint4 v;
    memcpy(&v, e, sizeof(v));
    *(uint4 *) p = v;
}

// tokens a warp takes: a lane writes 16 bytes at a time, so an f32 word of 8 channels takes two lanes (one lane with two
// 16-byte stores filled half sectors: 116 us instead of 77 for 50,000 rows of 8 heads of 128)
template <class T> __host__ __device__ constexpr int load_tokens() { return sizeof(T) == 4 ? 4 : 8; }

template <class T, int NG>
__global__ void __launch_bounds__(128) k_kv4_load(const Kv4Pool p, T * __restrict__ ko, T * __restrict__ vo,
                                                  const int64_t * __restrict__ slots, long long n) {
    constexpr int HD = 32 * NG, TOK = load_tokens<T>(), LANES = 32 / TOK, N = 16 / sizeof(T);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int lane = threadIdx.x & 31, t = lane % LANES / (LANES / 4), half = lane % (LANES / 4);
    const long long task = (long long) blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int h = (int) (task % p.heads);
    const long long tok = (task / p.heads) * TOK + lane / LANES;
    if (tok >= n) return;
    const long long slot = slots[tok];
    const bool live = slot >= 0 && slot < p.n_slots;
    const long long page = live ? slot >> p.page_shift : 0;
    const int at = live ? (int) (slot & ((1 << p.page_shift) - 1)) : 0, P = 1 << p.page_shift;
    const uint32_t * kq = (const uint32_t *) (p.q + kv4_q_at(p, page, 0, h, at)) + t * NG;
    const uint32_t * vq = (const uint32_t *) (p.q + kv4_q_at(p, page, 1, h, at)) + t;
    const __half * kd = p.d + kv4_d_at(p, page, 0, h, at);
    const __half * vd = p.d + kv4_d_at(p, page, 1, h, at);
    uint32_t kw[NG], vw[NG];
    float ks[NG], vs[NG];
#pragma unroll
    for (int g = 0; g < NG; g++) {
        kw[g] = kq[g];
        vw[g] = vq[4 * g];
        ks[g] = __half2float(kd[(size_t) g * P]);
        vs[g] = __half2float(vd[(size_t) g * P]);
    }
    const size_t o = ((size_t) tok * p.heads + h) * HD + 8 * t + 4 * half;
#pragma unroll
    for (int g = 0; g < NG; g++) write16<T, N>(ko + o + 32 * g, kw[g] >> (16 * half), ks[g], live);
#pragma unroll
    for (int g = 0; g < NG; g++) write16<T, N>(vo + o + 32 * g, vw[g] >> (16 * half), vs[g], live);
}

template <class T, int NG>
int store_launch(const Kv4Pool & p, const Kv4Rows & r, const int64_t * slots, long long n, dim3 grid, cudaStream_t st) {
    const long long strides = r.k_tok | r.k_head | r.v_tok | r.v_head;
    const bool vec = (((uintptr_t) r.k | (uintptr_t) r.v) & 15) == 0 && (strides * (long long) sizeof(T)) % 16 == 0;
    JB_CUDA(launch_pdl(k_kv4_store<T, NG>, grid, dim3(128), 0, st, p, r, slots, n, vec));
    return 0;
}
template <class T, int NG>
int load_launch(const Kv4Pool & p, const Kv4Rows & r, const int64_t * slots, long long n, dim3 grid, cudaStream_t st) {
    JB_CUDA(launch_pdl(k_kv4_load<T, NG>, grid, dim3(128), 0, st, p, (T *) r.k, (T *) r.v, slots, n));
    return 0;
}

template <class T>
int store_dim(const Kv4Pool & p, const Kv4Rows & r, const int64_t * slots, long long n, dim3 grid, cudaStream_t st) {
    switch (p.hd / 32) {
        case 1: return store_launch<T, 1>(p, r, slots, n, grid, st);
        case 2: return store_launch<T, 2>(p, r, slots, n, grid, st);
        case 3: return store_launch<T, 3>(p, r, slots, n, grid, st);
        default: return store_launch<T, 4>(p, r, slots, n, grid, st);
    }
}
template <class T>
int load_dim(const Kv4Pool & p, const Kv4Rows & r, const int64_t * slots, long long n, dim3 grid, cudaStream_t st) {
    switch (p.hd / 32) {
        case 1: return load_launch<T, 1>(p, r, slots, n, grid, st);
        case 2: return load_launch<T, 2>(p, r, slots, n, grid, st);
        case 3: return load_launch<T, 3>(p, r, slots, n, grid, st);
        default: return load_launch<T, 4>(p, r, slots, n, grid, st);
    }
}

double row_bytes(const Kv4Pool & p, int type) {
    return 2.0 * p.heads * p.hd * ((type == KV4_F32 ? 4 : 2) + 0.5625) + 8;
}

}  // namespace

int kv4_store(const Kv4Pool & p, const Kv4Rows & r, int type, const int64_t * slots, long long n, cudaStream_t st) {
    if (n < 1) return 0;
    const long long blocks = ((n + 7) / 8 * p.heads + 3) / 4;
    KTimer kt("kv4_store", st, 0, row_bytes(p, type) * n);
    const dim3 grid((unsigned) blocks);
    switch (type) {
        case KV4_F32: return store_dim<float>(p, r, slots, n, grid, st);
        case KV4_F16: return store_dim<__half>(p, r, slots, n, grid, st);
        default: return store_dim<__nv_bfloat16>(p, r, slots, n, grid, st);
    }
}

int kv4_load(const Kv4Pool & p, const Kv4Rows & r, int type, const int64_t * slots, long long n, cudaStream_t st) {
    if (n < 1) return 0;
    const int tok = type == KV4_F32 ? load_tokens<float>() : load_tokens<__half>();
    const long long blocks = ((n + tok - 1) / tok * p.heads + 3) / 4;
    KTimer kt("kv4_load", st, 0, row_bytes(p, type) * n);
    const dim3 grid((unsigned) blocks);
    switch (type) {
        case KV4_F32: return load_dim<float>(p, r, slots, n, grid, st);
        case KV4_F16: return load_dim<__half>(p, r, slots, n, grid, st);
        default: return load_dim<__nv_bfloat16>(p, r, slots, n, grid, st);
    }
}

// ------------------------------------------------------------------------------------------
// Block tables and slot maps of a step
// ------------------------------------------------------------------------------------------

namespace {

constexpr int TAB_THREADS = 512, TAB_RUN = 4;       // requests a thread takes at a time, in a row

struct Request { int cached, added, held, need, bad; };

__device__ __forceinline__ Request request_of(const KvTablesArgs & a, int r) {
    Request q = {0, 0, 0, 0, 0};
    if (r >= a.n_req) return q;
    q.cached = a.cached[r];
    q.added = a.added[r];
    const int P1 = (1 << a.page_shift) - 1;
    const long long len = (long long) q.cached + q.added;
    if (q.cached < 0 || q.added < 0) q.bad = 1;
    else if (len > (long long) a.width << a.page_shift || len > 0x7fffffffLL - P1) q.bad = 2;
    if (q.bad) { q.added = 0; return q; }
    q.held = (q.cached + P1) >> a.page_shift;
    q.need = (int) ((len + P1) >> a.page_shift) - q.held;
    return q;
}

// last index of v[0 .. n) (ascending, v[0] <= x) with v[i] <= x
__device__ __forceinline__ int last_le(const int * v, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (v[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
}

// Every CTA walks all requests, 4 a thread at a time: first their totals (in 64 bits), which decide whether the step is
// refused before anything is written, then a scan of new tokens and new pages, and writes its own share of the flat
// outputs: slots and fresh table entries, each found by bisection among the walked requests' first tokens / pages. One
// launch, no communication between CTAs, balanced however unequal the requests are; the lengths (8 bytes a
// request) stay in L2. 4000 requests and 517,000 slots in 148 CTAs: 13.7 us replayed (15 with cold caches; 8 walks of 512
// requests with two 64-bit scans took 22). The walk of 4000 requests alone takes 7.2 us, the 517,000 slots of 8 requests
// alone 6.7, 8 slots of 8 requests 2.9.
__global__ void __launch_bounds__(TAB_THREADS) k_kv_tables(const KvTablesArgs a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __shared__ int first_tok[TAB_THREADS * TAB_RUN], first_pg[TAB_THREADS * TAB_RUN], s_cached[TAB_THREADS * TAB_RUN];
    __shared__ long long w_tok[TAB_THREADS / 32], w_pg[TAB_THREADS / 32];
    __shared__ int2 w_sum[TAB_THREADS / 32];
    __shared__ int w_bad[TAB_THREADS / 32];
    const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5, nw = nt >> 5, run = nt * TAB_RUN;
    const int n_chunks = (a.n_req + run - 1) / run, P1 = (1 << a.page_shift) - 1;
    // totals and refusals; the first chunk's requests stay in registers
    Request q[TAB_RUN];
    long long tok = 0, pg = 0;
    int bad = 0x7fffffff;
#pragma unroll
    for (int k = 0; k < TAB_RUN; k++) q[k] = request_of(a, tid * TAB_RUN + k);
#pragma unroll
    for (int k = 0; k < TAB_RUN; k++) { tok += q[k].added; pg += q[k].need; if (q[k].bad) bad = min(bad, q[k].bad); }
    for (int c = 1; c < n_chunks; c++) {
#pragma unroll
        for (int k = 0; k < TAB_RUN; k++) {
            const Request o = request_of(a, c * run + tid * TAB_RUN + k);
            tok += o.added;
            pg += o.need;
            if (o.bad) bad = min(bad, o.bad);
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        tok += __shfl_xor_sync(0xffffffffu, tok, o);
        pg += __shfl_xor_sync(0xffffffffu, pg, o);
    }
    bad = __reduce_min_sync(0xffffffffu, bad);
    if (lane == 0) { w_tok[warp] = tok; w_pg[warp] = pg; w_bad[warp] = bad; }
    __syncthreads();
    tok = pg = 0;
    for (int w = 0; w < nw; w++) { tok += w_tok[w]; pg += w_pg[w]; bad = min(bad, w_bad[w]); }
    int status = bad == 0x7fffffff ? 0 : bad;
    if (!status && pg > a.n_free) status = 3;
    if (!status && tok > a.n_slots) status = 4;
    const int n_tok = status ? 0 : (int) tok, n_pg = status ? 0 : (int) pg;
    if (blockIdx.x == 0 && tid == 0) {
        a.state[0] = status;
        a.state[1] = n_pg;
        a.q_start[a.n_req] = n_tok;
    }
    const int s0 = (int) ((long long) a.n_slots * blockIdx.x / gridDim.x), s1 = (int) ((long long) a.n_slots * (blockIdx.x + 1) / gridDim.x);
    const int p0 = (int) ((long long) n_pg * blockIdx.x / gridDim.x), p1 = (int) ((long long) n_pg * (blockIdx.x + 1) / gridDim.x);
    for (int i = max(s0, n_tok) + tid; i < s1; i += nt) a.slots[i] = -1;
    int tok0 = 0, pg0 = 0;                // first token and page of the chunk (32 bits hold what is not refused)
    for (int c = 0; c < n_chunks; c++) {
        const int r0 = c * run, n = min(run, a.n_req - r0);
        const bool mine = c % gridDim.x == blockIdx.x;       // this CTA writes the chunk's lens and q_start
        if (status) {
            if (mine) {
                for (int i = tid; i < n; i += nt) { a.lens[r0 + i] = a.cached[r0 + i]; a.q_start[r0 + i] = 0; }
            }
            continue;
        }
        if (c) {
#pragma unroll
            for (int k = 0; k < TAB_RUN; k++) q[k] = request_of(a, r0 + tid * TAB_RUN + k);
        }
        int2 own = make_int2(0, 0);
#pragma unroll
        for (int k = 0; k < TAB_RUN; k++) { own.x += q[k].added; own.y += q[k].need; }
        int2 inc = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, inc.x, o), y = __shfl_up_sync(0xffffffffu, inc.y, o);
            if (lane >= o) { inc.x += x; inc.y += y; }
        }
        if (lane == 31) w_sum[warp] = inc;
        __syncthreads();
        int t = tok0 + inc.x - own.x, g = pg0 + inc.y - own.y, tok1 = tok0, pg1 = pg0;
        for (int w = 0; w < nw; w++) {
            const int2 s = w_sum[w];
            if (w < warp) { t += s.x; g += s.y; }
            tok1 += s.x;
            pg1 += s.y;
        }
#pragma unroll
        for (int k = 0; k < TAB_RUN; k++) {
            const int i = tid * TAB_RUN + k;
            first_tok[i] = t;
            first_pg[i] = g;
            s_cached[i] = q[k].cached;
            if (mine && i < n) { a.lens[r0 + i] = q[k].cached + q[k].added; a.q_start[r0 + i] = t; }
            t += q[k].added;
            g += q[k].need;
        }
        __syncthreads();
        for (int i = max(p0, pg0) + tid; i < min(p1, pg1); i += nt) {
            const int k = last_le(first_pg, n, i);
            a.table[(size_t) (r0 + k) * a.width + ((s_cached[k] + P1) >> a.page_shift) + (i - first_pg[k])] = a.free_pages[i];
        }
        for (int i = max(s0, tok0) + tid; i < min(s1, tok1); i += nt) {
            const int k = last_le(first_tok, n, i);
            const int pos = s_cached[k] + (i - first_tok[k]), idx = pos >> a.page_shift, held = (s_cached[k] + P1) >> a.page_shift;
            // a page held before this step comes from the table, a fresh one from the free list
            const int page = idx < held ? a.table[(size_t) (r0 + k) * a.width + idx] : a.free_pages[first_pg[k] + idx - held];
            a.slots[i] = page < 0 ? -1 : ((long long) page << a.page_shift) + (pos & P1);
        }
        tok0 = tok1;
        pg0 = pg1;
        __syncthreads();
    }
}

}  // namespace

int kv_tables(const KvTablesArgs & a, cudaStream_t st) {
    KTimer kt("kv_tables", st, 0, 16.0 * a.n_req + 8.0 * a.n_slots);
    // 4 slots a thread and more before another CTA joins; one CTA an SM at most (each walks every request)
    const int threads = a.n_req <= 128 && a.n_slots <= 512 ? 128 : TAB_THREADS;
    const int blocks = std::max(1, std::min(148, (a.n_slots + 4 * threads - 1) / (4 * threads)));
    JB_CUDA(launch_pdl(k_kv_tables, dim3((unsigned) blocks), dim3((unsigned) threads), 0, st, a));
    return 0;
}

}  // namespace jb
