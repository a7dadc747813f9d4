// jepa-b200 extensions: entry points this engine adds next to the jepa.cpp API (include/jepa.h).
//
// None of these replaces a reference function; they expose the engine's own pieces so that its kernels
// can be checked and timed through the same C ABI (plain pointers and sizes, host memory, int 0 / -1
// returns with the reason in jepa_error_text()), and so that a multi-GPU host can shard a planner.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include "jepa.h"

#ifdef __cplusplus
extern "C" {
#endif
#if defined(__GNUC__)
#pragma GCC visibility push(default)   // every declaration below is exported
#endif

// Version string of this engine ("jepa-b200 <version>").
const char * jepa_b200_version(void);

// C[M,N] = A[M,K] * B[N,K]^T on the current CUDA device through the tcgen05 3xTF32 GEMM of the planner
// (host buffers, row-major). A kernel check: the planner's linears all run through this kernel.
int jepa_b200_gemm(const float * A, const float * B, int M, int N, int K, float * C);

// The same product in the planner's configuration: narrow, long products (at most 8 output column tiles
// of 128, K >= 2048) split their K range in three parts whose partial tiles a fix-up sums in a fixed order (the
// planner passes that scratch on every such product). Agrees with jepa_b200_gemm to rounding.
int jepa_b200_gemm_ksplit(const float * A, const float * B, int M, int N, int K, float * C);

// The launch the planner's GEMM makes for a product of shape M x N x K, computed on the host (no device
// needed): out[0] = 1 for the persistent 128 x 128 kernel, 0 for the 64-wide split-K clusters; out[1] = the
// persistent kernel's K parts in the planner's configuration (1 = whole tiles; 0 for the clusters, whose split
// follows the device's cluster occupancy); out[2] = 1 when the persistent kernel walks grouped row tiles
// rows-fastest. A row's bits depend only on this plan, so rows of batches with the same plan agree bit for bit.
// Returns 0, or -1 for a null `out` or a non-positive size. No counterpart in the reference.
int jepa_b200_gemm_plan(int M, int N, int K, int * out);

// The persistent kernel's output tiles for that shape in the order its CTAs take them, computed on the host by
// the kernel's own tile-origin function: m0[t], n0[t] = first row and column of tile t. Returns the tile
// count, 0 when the shape takes the split-K clusters, -1 for null buffers, non-positive sizes or more than
// `cap` tiles. No counterpart in the reference.
int jepa_b200_gemm_tile_walk(int M, int N, int K, int * m0, int * n0, int cap);

// The planner-configuration product timed on the device: `reps` launches on device-resident operands,
// returns the mean milliseconds per launch in *ms (CUDA events around the launches).
int jepa_b200_gemm_bench(int M, int N, int K, int reps, double * ms);

// The planner's GEMM with its weight operand kept in GGUF block values and dequantised in the mainloop:
// W [rows][ne0] are the raw rows of a weight of ggml type 8 (q8_0), 2 (q4_0) or 1 (f16), rows and ne0
// multiples of 32. transposed = 0: C [M][rows] = A [M][ne0] W^T (the forward product); transposed = 1:
// C [M][ne0] = A [M][rows] W (the backward product against the same weight). ksplit = 1 passes the K-split
// scratch as the planner does. Equals jepa_b200_gemm on the dequantised weight bit for bit.
int jepa_b200_gemm_quant(uint32_t ggml_type, const void * w_raw, int rows, int ne0, int transposed, const float * A, int M,
                         float * C, int ksplit);

// jepa_b200_gemm_quant timed on the device (zero operands of shape M x N x K, `reps` launches); the mean
// milliseconds per launch in *ms.
int jepa_b200_gemm_quant_bench(uint32_t ggml_type, int M, int N, int K, int transposed, int reps, double * ms);

// jepa_b200_gemm for callers that must not allocate device memory. No counterpart in the reference.
// Some hosts cannot call cudaMalloc around a kernel call: a process whose device memory budget is fixed
// at start-up, a real-time control loop where an allocation (which can synchronise the whole device)
// would blow the cycle's deadline, or a plug-in living inside someone else's allocator. This entry point
// computes the same product as jepa_b200_gemm from the same host buffers, but keeps the device copies of
// A, B and C and the operand split planes in one fixed device array that the library reserves when it
// is loaded (JEPA_B200_NOALLOC_MAX_FLOATS floats = 16 MiB, held on every GPU that loads the library
// until the process exits), and calls no cudaMalloc / cudaFree.
//   limit  : 3 (M K + N K) + M N floats (each part rounded up to 64), at most JEPA_B200_NOALLOC_MAX_FLOATS;
//            larger sizes are refused with a message in jepa_error_text()
//   set-up : the first call on a device looks up that device's copy of the array, so make that first
//            call before any stream capture
//   sharing: every call on a device uses the same array and leaves its contents there; calls that
//            overlap on the GPU (from two host threads) race on it
// Runs on the current CUDA device and its legacy default stream; returns 0 or -1.
#define JEPA_B200_NOALLOC_MAX_FLOATS (4u * 1024u * 1024u)
int jepa_b200_gemm_noalloc(const float * A, const float * B, int M, int N, int K, float * C);

// The failure path of the engine's bounded device waits, run on purpose without a fault: one CTA takes
// tensor memory as the GEMM does, waits on an mbarrier that nothing arrives on with a bound of
// `limit_cycles` SM clock cycles (1 .. 4e9; the kernels' own bound is 4e9, about 2 s), raises the GEMM's
// error flag when the bound runs out, frees its tensor memory and returns. *code receives the flag as
// the engine reads it after a call (9 for this check, 0 if the wait did not run out); the read resets
// it. Returns 0 when the flag could be read and was reset, -1 otherwise. No counterpart in the reference
// (its planners run on the host and have no device waits).
int jepa_b200_check_wait_timeout(long long limit_cycles, int * code);

// The same rows decoded on the host by the loader's CPU decoder (no GPU needed): the decoder the engine
// uses for host-side tensors (recorded actions, the oracle's weights), checkable without a device.
int jepa_b200_host_dequant(uint32_t ggml_type, const void * src, int64_t rows, int64_t ne0, float * dst);

// Dequantise `rows` GGUF rows of `ne0` values of ggml type `ggml_type` (0 f32, 1 f16, 2 q4_0, 8 q8_0,
// 30 bf16) from the host bytes `src` into host float32 `dst` by the device kernel the weight loader uses.
int jepa_b200_dequant(uint32_t ggml_type, const void * src, int64_t rows, int64_t ne0, float * dst);

// Candidate sharding of the planners over `world` GPUs, one process (and one context) per GPU.
// Rank r plans candidates [r*S/world, (r+1)*S/world) of every level; the ranks exchange only each
// level's (min cost, index) and the winning plan, through NCCL over NVLink. `nccl_id` is the
// 128-byte ncclUniqueId from jepa_b200_nccl_unique_id() on rank 0, broadcast by the host.
// world == 1 turns sharding off. Must be called before the first planner call on `ctx`.
int jepa_b200_nccl_unique_id(void * out128);
int jepa_b200_context_set_shard(jepa_context * ctx, int rank, int world, const void * nccl_id);

// Device milliseconds of the last planner call on this context (CUDA events on its stream), and the
// number of kernels it launched.
double jepa_b200_last_plan_ms(const jepa_context * ctx);
long long jepa_b200_last_plan_launches(const jepa_context * ctx);

// Candidate streams of the H-JEPA solves on this context: a level's candidates (this GPU's share) run as
// n independent chains of consecutive rows side by side on the GPU (1..8; 0 = automatic: for predictors
// narrower than 768 one chain per 256 candidates, at most 4; for wider ones 2 from 512 candidates up, else 1).
// Results do not depend on n (rows never interact), as the reference's results do
// not depend on its thread count (its jepa_context_params.n_threads). Returns 0, or -1 for a non-H-JEPA
// context or n out of range.
int jepa_b200_hjepa_set_streams(jepa_context * ctx, int n);

// Memory mode of the H-JEPA solves on this context: 0 = automatic (the first that fits the free device memory
// of: every step's adaLN modulation and its gradient, [T S][6 P L] floats x 3; every step's modulation kept
// ([T S][6 P L] x 1) and the gradient folded step by step; one step at a time), 1 = always one step at a time
// (the modulation recomputed in the backward: more GEMM work, least memory), 2 = always the middle mode.
// Results are the same in every mode. Returns 0, or -1 for a non-H-JEPA context or a mode out of range.
int jepa_b200_hjepa_set_step_modulation(jepa_context * ctx, int mode);

// C[M,N] = f16(A)[M,K] * f16(B)[N,K]^T with f32 accumulation through the V-JEPA 2-AC predictor's
// tcgen05 kind::f16 GEMM (host f32 buffers, rounded to f16 on the device; K a multiple of 8). A kernel
// check: every linear of the AC predictor runs through this kernel.
int jepa_b200_gemm_f16(const float * A, const float * B, int M, int N, int K, float * C);
// Same product timed on device-resident operands: mean milliseconds per launch over `reps` launches.
int jepa_b200_gemm_f16_bench(int M, int N, int K, int reps, double * ms);

// The AC predictor's attention: the last of `n_frames` frames of `rows` rows attends to every row of all of
// them, for `n_cand` candidates and `heads` heads of width `hd` (16, 32 or 64). q [n_cand][rows][heads hd],
// kv [n_cand][n_frames rows][2 heads hd] (keys, then values), out like q: host f32, f16 on the device.
// impl: 0 the kernel the predictor would pick, 1 the mma.sync kernel, 2 the tcgen05 kernel (hd 64, rows <= 384).
int jepa_b200_attention(const float * q, const float * kv, int n_cand, int n_frames, int rows, int heads, int hd,
                        int impl, float * out);
// The same attention timed alone on pseudo-random device-resident f16 operands: mean milliseconds per launch.
int jepa_b200_attention_bench(int n_cand, int n_frames, int rows, int heads, int hd, int impl, int reps, double * ms);

// Per-kernel device timing for measurement runs. Between begin and end, every launch of the engine's
// instrumented kernels (the AC predictor's GEMM, attention and row kernels) in this process is bracketed
// by CUDA events on its stream. end() synchronises and writes one line per kernel kind into `out`
// ("<kind> <launches> <total ms> <algorithmic FLOPs> <algorithmic bytes>\n", at most cap bytes with the
// terminating 0) and returns the number of kinds (-1 if an event failed). The events cost a little
// overlap between neighbouring kernels, so time the headline numbers without it.
void jepa_b200_kprof_begin(void);
int jepa_b200_kprof_end(char * out, size_t cap);

// ---- A paged key / value cache held in 4 bits, for sessions of different lengths -------------------------------
//
// The entry points of this block work on DEVICE memory of the current device, on the caller's `stream` (a
// cudaStream_t; null = the legacy default stream), allocate nothing and do not synchronise, so they can be captured
// into a CUDA graph. They check their host arguments and that each pointer is memory of the current device; what lies
// in device memory (lengths, slots, page ids) is bounds-checked by the kernels. No counterpart in the reference.
//
// A pool of n_pages pages of page_size token rows; slot s is row s % page_size of page s / page_size. Layout:
//   q  uint8 [n_pages][2][kv_heads][page_size][head_dim / 2]   4-bit codes, low nibble first; plane 0 keys, 1 values
//   d  f16   [n_pages][2][kv_heads][head_dim / 32][page_size]  one scale per 32 channels of a row
// A code c stands for d (c - 8). Value rows keep their channels in order; a key row is a sequence of 8-channel words
// of which word t NG + g holds channels 32 g + 8 t .. + 7 (NG = head_dim / 32, t = 0 .. 3).
// 0.5625 bytes a value; both buffers must be 16-byte aligned (jepa_b200_kv4_bytes gives their sizes).
typedef struct jepa_b200_kv4_cache {
    void * q;
    void * d;
    int64_t n_pages;      // 1 .. 2^31 - 1
    int32_t page_size;    // 16, 32, 64, 128 or 256
    int32_t kv_heads;     // 1 .. 1024
    int32_t head_dim;     // 32, 64, 96 or 128
} jepa_b200_kv4_cache;

int jepa_b200_kv4_bytes(const jepa_b200_kv4_cache * cache, size_t * q_bytes, size_t * d_bytes);

// The bookkeeping of one step, built on the device: request r holds cached[r] tokens in the pages named by the first
// ceil(cached[r] / page_size) entries of its row of `table` [n_req][width], and gets added[r] more (0 is allowed).
// Fresh pages are taken from the start of free_pages [n_free], request by request, and written behind the held ones.
//   lens [n_req]          cached + added
//   q_start [n_req + 1]   exclusive sums of added: request r's new rows are q_start[r] .. q_start[r + 1] - 1
//   slots [n_slots]       the slot of every new row, in that order; -1 behind the last (and for a negative page id)
//   state [2]             {0, number of pages taken}, or {code, 0} of a refused step: 1 a negative length, 2 a request
//                         outgrows its table row (or 2^31), 3 too few free pages, 4 more than n_slots new rows
// A refused step (the smallest code of those that apply) leaves `table` as it was, sets lens = cached, q_start = 0 and
// slots = -1, so that the calls behind it store and compute nothing. Table entries behind the taken pages stay as
// they were. The arrays must not overlap. n_req, width, n_slots >= 1; n_req, n_slots, n_free <= 2^30.
int jepa_b200_kv_tables(const int32_t * cached, const int32_t * added, int n_req, int page_size, int32_t * table, int width,
                        const int32_t * free_pages, int n_free, int32_t * lens, int32_t * q_start, int64_t * slots, int n_slots,
                        int32_t * state, void * stream);

// Quantises n_tokens rows of keys and values into their slots. k, v: ggml type 0 (f32), 1 (f16) or 30 (bf16), element
// (token, head, channel) at token * tok + head * head_stride + channel (strides in elements). Per 32 channels: m = the
// value of largest magnitude (the positive one of two), d = m / -8 rounded to bf16, then f16, and clamped to +-8160;
// code = clamp(floor(x / d + 1/2) + 8, 0, 15), and 8 where d = 0. A group that holds an infinity or a NaN reads back as
// NaN. Rows whose slot is negative or behind the pool are skipped. The slots of one call must differ: of two rows with
// one slot, which one is kept is not defined (and may differ between groups).
int jepa_b200_kv4_store(const jepa_b200_kv4_cache * cache, const void * k, const void * v, uint32_t type, int64_t k_tok, int64_t k_head,
                        int64_t v_tok, int64_t v_head, const int64_t * slots, int64_t n_tokens, void * stream);

// Reads rows back: k, v [n_tokens][kv_heads][head_dim], contiguous and 16-byte aligned, of the given type (f16 and f32
// hold the cached values exactly; bf16 rounds them). A slot outside the pool reads as zeros; slots may repeat.
int jepa_b200_kv4_load(const jepa_b200_kv4_cache * cache, const int64_t * slots, int64_t n_tokens, void * k, void * v, uint32_t type,
                       void * stream);

// Attention of every request's new rows over its cached rows (the new ones among them: store first).
// Row i of the n = q_start[r + 1] - q_start[r] rows of request r stands at position p = lens[r] - n + i. It sees the
// keys j < lens[r]; with frame > 0 only those with j < (p / frame + 1) * frame (block-causal over frames of that many
// tokens; 1 = causal), and none when p < 0. A row that sees nothing gets zeros. Query heads are n_heads / kv_heads
// consecutive ones for each cache head. Rows of out outside every request's range are left as they were. A page id
// outside the pool leaves its keys out; lens is taken as at most width * page_size.
typedef struct jepa_b200_kv4_attn {
    const void * q;           // rows of `type`, element (row, head, channel) at row * q_tok + head * q_head + channel
    void * out;               // the same type, with its own strides; must not overlap q
    int64_t q_tok, q_head, o_tok, o_head;
    const int32_t * q_start;  // [n_req + 1], ascending from 0
    const int32_t * lens;     // [n_req]
    const int32_t * table;    // [n_req][width]
    int32_t n_req;            // 0 .. 65535
    int32_t n_rows;           // rows of q and out (n_rows * n_heads <= 2^30)
    int32_t width;
    int32_t n_heads;          // a multiple of kv_heads
    uint32_t type;            // 1 (f16) or 30 (bf16)
    int32_t frame;            // 0 = every cached key
    float scale;              // of the scores, usually 1 / sqrt(head_dim)
    int32_t max_len;          // bounds of lens and of rows per request that the launch is laid out for (0 = unknown):
    int32_t max_new;          // larger ones are computed all the same, with less of the GPU
    void * workspace;         // device, 16-byte aligned, jepa_b200_kv4_attention_workspace bytes; nothing is kept in
    size_t workspace_bytes;   // it between calls, but calls that may run at once need one each
} jepa_b200_kv4_attn;
int64_t jepa_b200_kv4_attention_workspace(const jepa_b200_kv4_cache * cache, const jepa_b200_kv4_attn * args);
// How that call is laid out, without making it: out[0] = 1 if many rows take the tiles kernel (0: all take the rows kernel),
// out[1] = CTAs along a cache head's columns, out[2] = key ranges, out[3] = keys of a range. 0, or -1 for bad arguments.
int jepa_b200_kv4_attention_plan(const jepa_b200_kv4_cache * cache, const jepa_b200_kv4_attn * args, int * out);
int jepa_b200_kv4_attention(const jepa_b200_kv4_cache * cache, const jepa_b200_kv4_attn * args, void * stream);

// Waits for `stream`, then reports the attention kernels of the current device, on whatever stream, that have given up one
// of their bounded waits since the last report: 0, or -1 with the reason (their unfinished rows are NaN). A failure is
// reported once, to whichever call comes first, so a program of several streams checks in one place, behind all of
// them. A capturing stream is refused.
int jepa_b200_kv4_check(void * stream);

// The same call with a failure made on purpose, for tests of what follows one: the kernel for many rows gives up at once
// at its wait `wait` (40 .. 51, the number that jepa_b200_kv4_check names), and at the others, which may then never be
// met, after limit_cycles (1 .. 4e9) clock cycles.
int jepa_b200_kv4_attention_giving_up(const jepa_b200_kv4_cache * cache, const jepa_b200_kv4_attn * args, int wait, long long limit_cycles,
                                      void * stream);

#if defined(__GNUC__)
#pragma GCC visibility pop
#endif
#ifdef __cplusplus
}
#endif
