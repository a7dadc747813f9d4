// Entry points of the paged 4-bit key / value cache (include/jepa_b200.h): argument checks, then the launchers of
// kv4.h. Every check that needs no device comes first, so a refusal is the same with and without one.
#include "kv4.h"
#include "common.h"
#include "../../include/jepa_b200.h"

#include <cmath>
#include <initializer_list>

using jb::log;

namespace {

struct Ptr { const char * name; const void * p; unsigned align; };

// every pointer non-null, aligned, and memory that the current device can reach as its own
int device_pointers(const char * fn, std::initializer_list<Ptr> ptrs) {
    for (const Ptr & q : ptrs) {
        if (!q.p) { log("jepa: %s: %s is null\n", fn, q.name); return -1; }
        if ((uintptr_t) q.p % q.align) { log("jepa: %s: %s must be %u-byte aligned\n", fn, q.name, q.align); return -1; }
    }
    int dev = 0;
    JB_CUDA(cudaGetDevice(&dev));
    for (const Ptr & q : ptrs) {
        cudaPointerAttributes at;
        JB_CUDA(cudaPointerGetAttributes(&at, q.p));
        if ((at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged) || (at.type == cudaMemoryTypeDevice && at.device != dev)) {
            log("jepa: %s: %s is not memory of the current device (%d)\n", fn, q.name, dev);
            return -1;
        }
    }
    return 0;
}

bool pool_of(const char * fn, const jepa_b200_kv4_cache * c, jb::Kv4Pool & p) {
    if (!c) { log("jepa: %s: the cache is null\n", fn); return false; }
    if (c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 96 && c->head_dim != 128) {
        log("jepa: %s: head_dim %d is not 32, 64, 96 or 128\n", fn, c->head_dim);
        return false;
    }
    if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1))) {
        log("jepa: %s: page_size %d is not 16, 32, 64, 128 or 256\n", fn, c->page_size);
        return false;
    }
    if (c->kv_heads < 1 || c->kv_heads > 1024 || c->n_pages < 1 || c->n_pages > 0x7fffffffLL) {
        log("jepa: %s: %lld pages of %d heads are out of range (1 .. 2^31 - 1 pages, 1 .. 1024 heads)\n", fn, (long long) c->n_pages, c->kv_heads);
        return false;
    }
    p.q = (uint8_t *) c->q;
    p.d = (__half *) c->d;
    p.page_shift = 0;
    while ((1 << p.page_shift) < c->page_size) p.page_shift++;
    p.n_slots = (long long) c->n_pages << p.page_shift;
    p.heads = c->kv_heads;
    p.hd = c->head_dim;
    return true;
}

// whether two of the rows x heads pieces of hd channels share an element; both strides are at least hd where they count
bool pieces_overlap(long long rows, long long tok, long long heads, long long head, int hd) {
    typedef __int128 wide;
    if (rows < 2 || heads < 2 || tok >= (wide) (heads - 1) * head + hd || head >= (wide) (rows - 1) * tok + hd) return false;
    // neither lies inside the other's steps: the closest rows to every head, from both sides
    for (long long h = 1; h < heads; h++) {
        const wide x = (wide) h * head, below = x / tok;
        for (wide r = below; r <= below + 1; r++) {
            const wide gap = r * tok - x;
            if (r >= 1 && r < rows && gap < hd && gap > -hd) return true;
        }
    }
    return false;
}

bool attn_of(const char * fn, const jb::Kv4Pool & p, const jepa_b200_kv4_attn * x, jb::Kv4Attn & a) {
    if (!x) { log("jepa: %s: the arguments are null\n", fn); return false; }
    if (x->type != jb::KV4_F16 && x->type != jb::KV4_BF16) { log("jepa: %s: type %u is not 1 (f16) or 30 (bf16)\n", fn, x->type); return false; }
    if (x->n_heads < 1 || x->n_heads > 65535 || x->n_heads % p.heads) {
        log("jepa: %s: %d query heads are not a multiple of the cache's %d, or more than 65535\n", fn, x->n_heads, p.heads);
        return false;
    }
    if (x->n_req < 0 || x->n_req > 65535 || x->n_rows < 0 || x->width < 1) {
        log("jepa: %s: %d requests (0 .. 65535), %d rows, %d table columns are out of range\n", fn, x->n_req, x->n_rows, x->width);
        return false;
    }
    if (((long long) x->width << p.page_shift) > 0x7fffffffLL - 1024) { log("jepa: %s: %d table columns exceed 2^31 positions\n", fn, x->width); return false; }
    if ((long long) x->n_rows * x->n_heads > (1 << 30)) { log("jepa: %s: %d rows of %d heads are more than 2^30\n", fn, x->n_rows, x->n_heads); return false; }
    if (x->frame < 0 || x->max_len < 0 || x->max_new < 0) { log("jepa: %s: frame %d, max_len %d and max_new %d must not be negative\n", fn, x->frame, x->max_len, x->max_new); return false; }
    if (!std::isfinite(x->scale)) { log("jepa: %s: scale is not finite\n", fn); return false; }
    if (x->q_tok < 0 || x->q_head < 0 || x->o_tok < 0 || x->o_head < 0) { log("jepa: %s: strides must not be negative\n", fn); return false; }
    if (x->n_rows > 1 && x->o_tok < p.hd) { log("jepa: %s: rows of out overlap (stride %lld of %d channels)\n", fn, (long long) x->o_tok, p.hd); return false; }
    if (x->n_heads > 1 && x->o_head < p.hd) { log("jepa: %s: heads of out overlap (stride %lld of %d channels)\n", fn, (long long) x->o_head, p.hd); return false; }
    if (pieces_overlap(x->n_rows, x->o_tok, x->n_heads, x->o_head, p.hd)) {
        log("jepa: %s: rows and heads of out overlap (strides %lld and %lld)\n", fn, (long long) x->o_tok, (long long) x->o_head);
        return false;
    }
    a.q = x->q; a.out = x->out;
    a.q_tok = x->q_tok; a.q_head = x->q_head; a.o_tok = x->o_tok; a.o_head = x->o_head;
    a.q_start = x->q_start; a.lens = x->lens; a.table = x->table;
    a.n_req = x->n_req; a.width = x->width; a.heads = x->n_heads; a.n_rows = x->n_rows;
    a.frame = x->frame; a.scale = x->scale; a.type = (int) x->type;
    // the longest context and the most rows of one request, as far as the caller can say: they shape the launch only
    const long long cap = (long long) x->width << p.page_shift;
    a.max_len = (int) (x->max_len < 1 || x->max_len > cap ? cap : x->max_len);
    a.max_new = x->max_new < 1 || x->max_new > x->n_rows ? x->n_rows : x->max_new;
    a.ws = x->workspace; a.ws_bytes = x->workspace_bytes;
    return true;
}

bool row_type(const char * fn, uint32_t type) {
    if (type == jb::KV4_F32 || type == jb::KV4_F16 || type == jb::KV4_BF16) return true;
    log("jepa: %s: type %u is not 0 (f32), 1 (f16) or 30 (bf16)\n", fn, type);
    return false;
}

int attention(const char * fn, const jepa_b200_kv4_cache * cache, const jepa_b200_kv4_attn * args, const jb::Kv4Waits & waits, void * stream) {
    jb::Kv4Pool p;
    jb::Kv4Attn a;
    if (!pool_of(fn, cache, p) || !attn_of(fn, p, args, a)) return -1;
    if (!a.n_req || !a.n_rows) return 0;
    const size_t need = jb::kv4_attention_workspace(p, a);
    if (a.ws_bytes < need) {
        log("jepa: %s: the workspace holds %zu bytes, this call needs %zu\n", fn, a.ws_bytes, need);
        return -1;
    }
    const void * ws = need ? a.ws : p.q;
    if (device_pointers(fn, {{"cache.q", p.q, 16}, {"cache.d", p.d, 16}, {"q", a.q, 2}, {"out", a.out, 2}, {"q_start", a.q_start, 4},
                             {"lens", a.lens, 4}, {"table", a.table, 4}, {"workspace", ws, 16}})) return -1;
    return jb::kv4_attention(p, a, waits, (cudaStream_t) stream);
}

// tokens of a store or load: a block takes 16 (token, head) pairs at least, and a grid has 2^31 - 1 blocks
bool token_count(const char * fn, const jb::Kv4Pool & p, int64_t n) {
    const int64_t most = (0x7fffffffLL / p.heads - 1) * 16;
    if (n >= 0 && n <= most) return true;
    log("jepa: %s: %lld tokens are out of range (0 .. %lld for %d heads)\n", fn, (long long) n, (long long) most, p.heads);
    return false;
}

}  // namespace

extern "C" {

int jepa_b200_kv4_bytes(const jepa_b200_kv4_cache * cache, size_t * q_bytes, size_t * d_bytes) {
    jb::Kv4Pool p;
    if (!pool_of("jepa_b200_kv4_bytes", cache, p)) return -1;
    if (!q_bytes || !d_bytes) { log("jepa: jepa_b200_kv4_bytes: the results' pointers are null\n"); return -1; }
    *q_bytes = jb::kv4_q_at(p, cache->n_pages, 0, 0, 0);
    *d_bytes = jb::kv4_d_at(p, cache->n_pages, 0, 0, 0) * sizeof(__half);
    return 0;
}

int jepa_b200_kv_tables(const int32_t * cached, const int32_t * added, int n_req, int page_size, int32_t * table, int width,
                        const int32_t * free_pages, int n_free, int32_t * lens, int32_t * q_start, int64_t * slots, int n_slots,
                        int32_t * state, void * stream) {
    static const char * fn = "jepa_b200_kv_tables";
    constexpr int MAX = 1 << 30;        // of each count: the kernel's 32-bit indices step past the end by less than that
    if (n_req < 1 || width < 1 || n_free < 0 || n_slots < 1 || n_req > MAX || n_free > MAX || n_slots > MAX) {
        log("jepa: %s: need n_req, width and n_slots of 1 or more, n_free of 0 or more, none above 2^30 (%d, %d, %d, %d)\n", fn, n_req, width, n_slots, n_free);
        return -1;
    }
    if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1))) {
        log("jepa: %s: page_size %d is not 16, 32, 64, 128 or 256\n", fn, page_size);
        return -1;
    }
    const void * fp = n_free ? (const void *) free_pages : (const void *) table;   // no page to give: never read
    if (device_pointers(fn, {{"cached", cached, 4}, {"added", added, 4}, {"table", table, 4}, {"free_pages", fp, 4}, {"lens", lens, 4},
                             {"q_start", q_start, 4}, {"slots", slots, 8}, {"state", state, 4}})) return -1;
    jb::KvTablesArgs a{cached, added, n_req, 0, table, width, (const int32_t *) fp, n_free, lens, q_start, slots, n_slots, state};
    while ((1 << a.page_shift) < page_size) a.page_shift++;
    return jb::kv_tables(a, (cudaStream_t) stream);
}

int jepa_b200_kv4_store(const jepa_b200_kv4_cache * cache, const void * k, const void * v, uint32_t type, int64_t k_tok, int64_t k_head,
                        int64_t v_tok, int64_t v_head, const int64_t * slots, int64_t n_tokens, void * stream) {
    static const char * fn = "jepa_b200_kv4_store";
    jb::Kv4Pool p;
    if (!pool_of(fn, cache, p) || !row_type(fn, type)) return -1;
    if (!token_count(fn, p, n_tokens)) return -1;
    if (k_tok < 0 || k_head < 0 || v_tok < 0 || v_head < 0) { log("jepa: %s: strides must not be negative\n", fn); return -1; }
    if (!n_tokens) return 0;
    const unsigned size = type == jb::KV4_F32 ? 4 : 2;
    if (device_pointers(fn, {{"cache.q", p.q, 16}, {"cache.d", p.d, 16}, {"k", k, size}, {"v", v, size}, {"slots", slots, 8}})) return -1;
    return jb::kv4_store(p, {(void *) k, (void *) v, k_tok, k_head, v_tok, v_head}, (int) type, slots, n_tokens, (cudaStream_t) stream);
}

int jepa_b200_kv4_load(const jepa_b200_kv4_cache * cache, const int64_t * slots, int64_t n_tokens, void * k, void * v, uint32_t type,
                       void * stream) {
    static const char * fn = "jepa_b200_kv4_load";
    jb::Kv4Pool p;
    if (!pool_of(fn, cache, p) || !row_type(fn, type)) return -1;
    if (!token_count(fn, p, n_tokens)) return -1;
    if (!n_tokens) return 0;
    if (device_pointers(fn, {{"cache.q", p.q, 16}, {"cache.d", p.d, 16}, {"k", k, 16}, {"v", v, 16}, {"slots", slots, 8}})) return -1;
    return jb::kv4_load(p, {k, v, 0, 0, 0, 0}, (int) type, slots, n_tokens, (cudaStream_t) stream);
}

int64_t jepa_b200_kv4_attention_workspace(const jepa_b200_kv4_cache * cache, const jepa_b200_kv4_attn * args) {
    static const char * fn = "jepa_b200_kv4_attention_workspace";
    jb::Kv4Pool p;
    jb::Kv4Attn a;
    if (!pool_of(fn, cache, p) || !attn_of(fn, p, args, a)) return -1;
    return (int64_t) jb::kv4_attention_workspace(p, a);
}

int jepa_b200_kv4_attention_plan(const jepa_b200_kv4_cache * cache, const jepa_b200_kv4_attn * args, int * out) {
    static const char * fn = "jepa_b200_kv4_attention_plan";
    jb::Kv4Pool p;
    jb::Kv4Attn a;
    if (!pool_of(fn, cache, p) || !attn_of(fn, p, args, a)) return -1;
    if (!out || !a.n_req || !a.n_rows) { log("jepa: %s: needs a result's pointer, requests and rows\n", fn); return -1; }
    jb::kv4_attention_plan(p, a, out);
    return 0;
}

int jepa_b200_kv4_attention(const jepa_b200_kv4_cache * cache, const jepa_b200_kv4_attn * args, void * stream) {
    return attention("jepa_b200_kv4_attention", cache, args, jb::Kv4Waits(), stream);
}

int jepa_b200_kv4_attention_giving_up(const jepa_b200_kv4_cache * cache, const jepa_b200_kv4_attn * args, int wait, long long limit_cycles,
                                      void * stream) {
    static const char * fn = "jepa_b200_kv4_attention_giving_up";
    if (wait < 40 || wait > 51 || limit_cycles < 1 || limit_cycles > 4000000000LL) {
        log("jepa: %s: need 40 <= wait <= 51 and 1 <= limit_cycles <= 4e9 (%d, %lld)\n", fn, wait, limit_cycles);
        return -1;
    }
    jb::Kv4Waits waits;
    waits.limit = limit_cycles;
    waits.give_up_at = wait;
    return attention(fn, cache, args, waits, stream);
}

int jepa_b200_kv4_check(void * stream) {
    cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
    JB_CUDA(cudaStreamIsCapturing((cudaStream_t) stream, &capturing));
    if (capturing != cudaStreamCaptureStatusNone) { log("jepa: jepa_b200_kv4_check: the stream is capturing\n"); return -1; }
    const int code = jb::kv4_error_flag((cudaStream_t) stream);
    if (code > 0) log("jepa: jepa_b200_kv4_check: an attention kernel gave up waiting on its pipeline (wait %d); the rows that it had not finished are NaN\n", code);
    return code == 0 ? 0 : -1;
}

}  // extern "C"
