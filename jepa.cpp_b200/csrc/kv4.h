// The paged key / value cache held in 4 bits: layout, argument blocks and launchers (kv4.cu, kv4_attention.cu;
// checks and entry points in kv4_api.cpp).
//
// A pool of n_pages pages of P token rows; slot s is row s % P of page s / P.
//   q  4-bit codes, low nibble first      [n_pages][2][H][P][hd / 2]       (plane 0 keys, plane 1 values)
//   d  f16 scales, one per 32 channels    [n_pages][2][H][hd / 32][P]
// A code c stands for d (c - 8), the arithmetic of a q4_0 block. d is kept to 8 significant bits, so that
// d (c - 8) has at most 11 and is exact in f16: attention feeds the tensor cores the cached values themselves.
// A row is read as 8-channel words (4 bytes). Value rows keep their channels in order. Key rows interleave the
// words of their 32-channel groups, word t NG + g = channels 32 g + 8 t .. + 7 (NG = hd / 32): a lane that needs 8
// channels of every group for a k-step finds them side by side.
#pragma once

#include <cuda_runtime.h>
#include <cuda_fp16.h>
#include <cstddef>
#include <cstdint>

namespace jb {

struct Kv4Pool {
    uint8_t * q = nullptr;
    __half * d = nullptr;
    long long n_slots = 0;          // n_pages * P
    int page_shift = 0;             // P = 1 << page_shift
    int heads = 0, hd = 0;
};

// first byte of row `row` (0 .. P - 1) of head h of a plane, and the index of its first scale (group g: + g * P)
__host__ __device__ inline size_t kv4_q_at(const Kv4Pool & p, long long page, int plane, int h, int row) {
    return (((((size_t) page * 2 + plane) * p.heads + h) << p.page_shift) + row) * (size_t) (p.hd / 2);
}
__host__ __device__ inline size_t kv4_d_at(const Kv4Pool & p, long long page, int plane, int h, int row) {
    return (((((size_t) page * 2 + plane) * p.heads + h) * (size_t) (p.hd / 32)) << p.page_shift) + row;
}

enum Kv4Type : int { KV4_F32 = 0, KV4_F16 = 1, KV4_BF16 = 30 };   // ggml type numbers, as in the loader

struct Kv4Rows {                    // k and v rows of n tokens, strides in elements, channels contiguous
    void * k = nullptr, * v = nullptr;
    long long k_tok = 0, k_head = 0, v_tok = 0, v_head = 0;
};

int kv4_store(const Kv4Pool & p, const Kv4Rows & r, int type, const int64_t * slots, long long n, cudaStream_t st);
int kv4_load(const Kv4Pool & p, const Kv4Rows & r, int type, const int64_t * slots, long long n, cudaStream_t st);

struct KvTablesArgs {
    const int32_t * cached, * added;
    int n_req, page_shift;
    int32_t * table;
    int width;
    const int32_t * free_pages;
    int n_free;
    int32_t * lens, * q_start;
    int64_t * slots;
    int n_slots;
    int32_t * state;
};
int kv_tables(const KvTablesArgs & a, cudaStream_t st);

struct Kv4Attn {
    const void * q;
    void * out;
    long long q_tok, q_head, o_tok, o_head;
    const int32_t * q_start, * lens, * table;
    int n_req, width, heads, n_rows;    // n_rows: rows of q (and out)
    int frame;
    float scale;
    int max_len, max_new;
    int type;
    void * ws;
    size_t ws_bytes;
};
// the bounded waits of the tiles kernel
struct Kv4Waits {
    long long limit = 4000000000LL;         // cycles before one gives up (about 2 s)
    int give_up_at = 0;                     // the one (by its code) that gives up at once: the failure path's test
};
size_t kv4_attention_workspace(const Kv4Pool & p, const Kv4Attn & a);
void kv4_attention_plan(const Kv4Pool & p, const Kv4Attn & a, int * out);      // see jepa_b200_kv4_attention_plan
int kv4_attention(const Kv4Pool & p, const Kv4Attn & a, const Kv4Waits & w, cudaStream_t st);
// Waits for the stream: the wait that ran out in a kernel of the current device, if one did that no call has told yet; 0, or -1: not read
int kv4_error_flag(cudaStream_t st);

}  // namespace jb
