// C ABI, part 5: the paged key-value cache - tables, append and attention over one pool of pages on the caller's device memory.
// Every check is made before anything is enqueued; the calls never synchronise, allocate or keep a workspace, so they can be captured.
#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <new>

#include "../../include/aha_amd.h"
#include "paged.h"

struct aha_paged {
    aha_paged_desc d;
    int device, lps;
    std::atomic<int> n_cus;                      // asked for once, by the first attention call
    std::atomic<int> precise;
};

static thread_local char g_paged_err[256];
static int refuse(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_paged_err, sizeof(g_paged_err), fmt, ap);
    va_end(ap);
    return code;
}
enum { E_INVAL = -22, E_NOMEM = -12, E_HIP = -5, E_RANGE = -34 };

// the pool's device for the duration of a call, whatever the caller's current one is
struct OnDevice {
    int was = -1, now;
    hipError_t err;
    explicit OnDevice(int device) : now(device) {
        err = hipGetDevice(&was);
        if (err == hipSuccess && was != device) err = hipSetDevice(device);
    }
    ~OnDevice() { if (was >= 0 && was != now) (void)hipSetDevice(was); }
};
#define RUN(what, expr)                                                                                          \
    do {                                                                                                         \
        OnDevice on_(p->device);                                                                                 \
        hipError_t e_ = on_.err;                                                                                 \
        if (e_ == hipSuccess) e_ = (expr);                                                                       \
        if (e_ != hipSuccess) return refuse(E_HIP, what ": %s", hipGetErrorString(e_));                          \
    } while (0)

static bool aligned16(const void* x) { return ((uintptr_t)x & 15) == 0; }

// Do rows of `a` (n of them, wa elements each, lda apart) and of `b` share an element?  Rows of one buffer may lie between each other (the columns of a
// fused projection) if they have the same stride; with another one, ranges that meet are taken to.
static bool rows_meet(const void* a, int64_t lda, int64_t wa, const void* b, int64_t ldb, int64_t wb, int64_t n) {
    const int64_t x = (intptr_t)a / 2, y = (intptr_t)b / 2;               // (bf16 elements; addresses are below 2^63)
    if (x + (n - 1) * lda + wa <= y || y + (n - 1) * ldb + wb <= x) return false;
    if (n == 1 || lda != ldb) return true;
    const int64_t off = ((y - x) % lda + lda) % lda;
    return off < wa || off + wb > lda;
}

extern "C" const char* aha_paged_last_error(void) { return g_paged_err; }

extern "C" int aha_paged_create(const aha_paged_desc* d, int device, aha_paged** out) {
    if (!d || !out || device < 0) return refuse(E_INVAL, "null argument or negative device");
    if (!d->k_pages || !d->v_pages || !d->block_table || !d->lens || !d->free_pages || !d->n_free) return refuse(E_INVAL, "null tensor");
    if (!aligned16(d->k_pages) || !aligned16(d->v_pages)) return refuse(E_INVAL, "pages must be aligned to 16 bytes");
    if (d->kv_type != AHA_KV_BF16 && d->kv_type != AHA_KV_E4M3) return refuse(E_INVAL, "unknown kv_type %d", d->kv_type);
    if (d->kv_type == AHA_KV_BF16 && (d->k_scale || d->v_scale)) return refuse(E_INVAL, "scales belong to an 8-bit cache");
    if (d->layers < 1 || d->n_pages < 1 || d->max_blocks < 1) return refuse(E_INVAL, "layers, n_pages and max_blocks must be positive");
    if (d->max_seqs < 1 || d->max_seqs > PAGED_MAX_SEQS) return refuse(E_RANGE, "max_seqs must be 1..%d", PAGED_MAX_SEQS);
    if (d->kv_heads < 1 || d->kv_heads > 1024) return refuse(E_RANGE, "kv_heads must be 1..1024");
    if (d->head_dim < 16 || d->head_dim > 128 || d->head_dim % 16) return refuse(E_RANGE, "head_dim must be a multiple of 16, at most 128");
    if (d->page_size < 16 || d->page_size > 1024 || (d->page_size & (d->page_size - 1))) return refuse(E_RANGE, "page_size must be a power of two, 16..1024");
    if ((int64_t)d->n_pages * d->page_size > 0x7fffffff) return refuse(E_RANGE, "more than 2^31 - 1 slots");
    if ((int64_t)d->max_blocks * d->page_size > 0x7fffffff - 4096) return refuse(E_RANGE, "sequences of more than 2^31 - 4097 tokens");
    aha_paged* p = new (std::nothrow) aha_paged();
    if (!p) return refuse(E_NOMEM, "out of memory");
    p->d = *d; p->device = device; p->lps = 0; p->n_cus = 0; p->precise = 0;
    while ((1 << p->lps) < d->page_size) ++p->lps;
    *out = p;
    return 0;
}
extern "C" int aha_paged_set_precise(aha_paged* p, int on) {
    if (!p) return refuse(E_INVAL, "null handle");
    p->precise = on != 0;
    return 0;
}
extern "C" void aha_paged_destroy(aha_paged* p) { delete p; }

static PagedTables tables_of(const aha_paged* p) {
    return {p->d.block_table, p->d.lens, p->d.free_pages, p->d.n_free, p->d.n_pages, p->lps, p->d.max_seqs, p->d.max_blocks};
}
extern "C" int aha_paged_reserve(aha_paged* p, const int32_t* seqs, const int32_t* counts, int n, int32_t* slots, int32_t* positions, int n_tokens,
                                 int32_t* cu_tokens, int32_t* status, aha_hip_stream st) {
    if (!p || !cu_tokens || !status) return refuse(E_INVAL, "null argument");
    if (n < 0 || n_tokens < 0 || (n && (!seqs || !counts)) || (n_tokens && (!slots || !positions))) return refuse(E_INVAL, "null array or negative size");
    if (n > 2 * PAGED_MAX_SEQS) return refuse(E_RANGE, "more than %d requests", 2 * PAGED_MAX_SEQS);
    if (n_tokens > 0x7fffffff - 4096) return refuse(E_RANGE, "too many tokens in one call");
    PagedReserveArgs a = {tables_of(p), seqs, counts, n, slots, positions, n_tokens, cu_tokens, status};
    RUN("paged reserve", paged_reserve(&a, (hipStream_t)st));
    return 0;
}
extern "C" int aha_paged_truncate(aha_paged* p, const int32_t* seqs, const int32_t* new_lens, int n, int32_t* status, aha_hip_stream st) {
    if (!p || !status || n < 0 || (n && (!seqs || !new_lens))) return refuse(E_INVAL, "null argument or negative size");
    if (n > 2 * PAGED_MAX_SEQS) return refuse(E_RANGE, "more than %d requests", 2 * PAGED_MAX_SEQS);
    PagedReserveArgs a = {tables_of(p), seqs, new_lens, n, nullptr, nullptr, 0, nullptr, status};
    RUN("paged truncate", paged_truncate(&a, (hipStream_t)st));
    return 0;
}

static size_t layer_bytes(const aha_paged_desc& d) {
    return (size_t)d.n_pages * d.kv_heads * d.page_size * d.head_dim * (d.kv_type == AHA_KV_BF16 ? 2 : 1);
}
extern "C" int aha_paged_append(aha_paged* p, int layer, const void* q, int64_t ldq, int heads, void* q_out, int64_t ldqo, const void* k, int64_t ldk,
                                const void* v, int64_t ldv, const int32_t* slots, const int32_t* positions, int n_tokens, const void* cos,
                                const void* sin, int n_pos, aha_hip_stream st) {
    if (!p || n_tokens < 0 || heads < 0) return refuse(E_INVAL, "null handle or negative size");
    if (n_tokens == 0) return 0;
    const aha_paged_desc& d = p->d;
    if (!k || !v || !slots || (heads && (!q || !q_out))) return refuse(E_INVAL, "null tensor");
    if (layer < 0 || layer >= d.layers) return refuse(E_RANGE, "layer out of range");
    if (heads > 4096) return refuse(E_RANGE, "heads must be at most 4096");
    if ((cos != nullptr) != (sin != nullptr) || (cos && (!positions || n_pos < 1))) return refuse(E_INVAL, "rotation needs cos, sin, n_pos and positions");
    const int64_t qw = (int64_t)heads * d.head_dim, kw = (int64_t)d.kv_heads * d.head_dim;
    if (ldk < kw || ldv < kw || (heads && (ldq < qw || ldqo < qw))) return refuse(E_RANGE, "a row stride is shorter than its row");
    if (ldk % 8 || ldv % 8 || (heads && (ldq % 8 || ldqo % 8))) return refuse(E_RANGE, "row strides must be multiples of 8 elements");
    if (!aligned16(k) || !aligned16(v) || !aligned16(cos) || !aligned16(sin) || (heads && (!aligned16(q) || !aligned16(q_out))))
        return refuse(E_INVAL, "tensors must be aligned to 16 bytes");
    if (heads && (q == q_out ? n_tokens > 1 && ldq != ldqo : rows_meet(q, ldq, qw, q_out, ldqo, qw, n_tokens)))
        return refuse(E_INVAL, "q_out overlaps q: it must be q itself, ldq and ldqo equal, or lie elsewhere");
    if (heads && (rows_meet(k, ldk, kw, q_out, ldqo, qw, n_tokens) || rows_meet(v, ldv, kw, q_out, ldqo, qw, n_tokens)))
        return refuse(E_INVAL, "q_out overlaps k or v");
    if ((int64_t)n_tokens * (heads + 2 * d.kv_heads) * (d.head_dim / 16) > 0x7fffffff) return refuse(E_RANGE, "too many tokens in one call");
    PagedAppendArgs a;
    a.q = (const bf16*)q; a.k = (const bf16*)k; a.v = (const bf16*)v; a.ldq = ldq; a.ldk = ldk; a.ldv = ldv;
    a.q_out = (bf16*)q_out; a.ldqo = ldqo;
    a.k_pages = (char*)d.k_pages + layer * layer_bytes(d); a.v_pages = (char*)d.v_pages + layer * layer_bytes(d);
    a.k_scale = d.k_scale ? d.k_scale + (size_t)layer * d.kv_heads : nullptr;
    a.v_scale = d.v_scale ? d.v_scale + (size_t)layer * d.kv_heads : nullptr;
    a.slots = slots; a.positions = positions; a.cos = (const bf16*)cos; a.sin = (const bf16*)sin; a.n_pos = n_pos;
    a.n_tokens = n_tokens; a.heads = heads; a.kv_heads = d.kv_heads; a.hd = d.head_dim; a.lps = p->lps; a.n_slots = d.n_pages * d.page_size;
    a.e4m3 = d.kv_type == AHA_KV_E4M3;
    RUN("paged append", paged_append(&a, (hipStream_t)st));
    return 0;
}

static int cus_of(aha_paged* p, int* out) {
    int n = p->n_cus;
    if (!n) {
        RUN("compute units", hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, p->device));
        p->n_cus = n;
    }
    *out = n;
    return 0;
}
static int attention_sizes(const aha_paged* p, int heads, int n_tokens, int n, int max_q, int max_len) {
    const aha_paged_desc& d = p->d;
    if (n_tokens < 0 || n < 0 || max_q < 0 || max_len < 0) return refuse(E_INVAL, "negative size");
    if (heads < 1 || heads > 4096 || heads % d.kv_heads) return refuse(E_RANGE, "heads must be a multiple of the cache's key-value heads, at most 4096");
    if (n > 2 * PAGED_MAX_SEQS) return refuse(E_RANGE, "more than %d requests", 2 * PAGED_MAX_SEQS);
    if ((int64_t)n_tokens * heads > 0xffffff || (int64_t)n * d.kv_heads > 0x7fffff) return refuse(E_RANGE, "too many tokens or requests in one call");
    return 0;
}
static int attention_plan(aha_paged* p, int heads, int n_tokens, int n, int max_q, int max_len, PagedAttnArgs* a, size_t* bytes) {
    const aha_paged_desc& d = p->d;
    a->n = n; a->n_tokens = n_tokens; a->max_seqs = d.max_seqs; a->max_blocks = d.max_blocks; a->n_pages = d.n_pages; a->lps = p->lps;
    a->kv_heads = d.kv_heads; a->G = heads / d.kv_heads; a->hd = d.head_dim;
    int cus;
    if (int rc = cus_of(p, &cus)) return rc;
    *bytes = paged_attention_plan(a, cus, max_q, max_len);
    return 0;
}
extern "C" int aha_paged_attention_workspace(aha_paged* p, int heads, int n_tokens, int n, int max_q, int max_len, size_t* bytes) {
    if (!p || !bytes) return refuse(E_INVAL, "null argument");
    if (int rc = attention_sizes(p, heads, n_tokens, n, max_q, max_len)) return rc;
    PagedAttnArgs a;
    return attention_plan(p, heads, n_tokens, n, max_q, max_len, &a, bytes);
}
extern "C" int aha_paged_attention(aha_paged* p, int layer, const void* q, int64_t ldq, int heads, const int32_t* seqs, const int32_t* cu_tokens,
                                   int n, int n_tokens, int max_q, int max_len, int window, float scale, void* out, int64_t ldo, void* workspace,
                                   size_t workspace_bytes, aha_hip_stream st) {
    if (!p) return refuse(E_INVAL, "null handle");
    const aha_paged_desc& d = p->d;
    if (layer < 0 || layer >= d.layers) return refuse(E_RANGE, "layer out of range");
    if (window < 0) return refuse(E_INVAL, "negative window");
    if (!(scale > 0.f) || scale > 3e38f) return refuse(E_INVAL, "scale must be positive and finite");
    if (int rc = attention_sizes(p, heads, n_tokens, n, max_q, max_len)) return rc;
    if (n_tokens == 0 || n == 0) return 0;
    if (!q || !out || !seqs || !cu_tokens) return refuse(E_INVAL, "null tensor");
    const int64_t qw = (int64_t)heads * d.head_dim;
    if (ldq < qw || ldo < qw || ldq % 8 || ldo % 8) return refuse(E_RANGE, "row strides must hold a row and be multiples of 8 elements");
    if (!aligned16(q) || !aligned16(out) || !aligned16(workspace)) return refuse(E_INVAL, "tensors must be aligned to 16 bytes");
    if (q == out ? n_tokens > 1 && ldq != ldo : rows_meet(q, ldq, qw, out, ldo, qw, n_tokens))
        return refuse(E_INVAL, "out overlaps q: it must be q itself, ldq and ldo equal, or lie elsewhere");
    PagedAttnArgs a;
    size_t need = 0;
    if (int rc = attention_plan(p, heads, n_tokens, n, max_q, max_len, &a, &need)) return rc;
    if (need && (!workspace || workspace_bytes < need)) return refuse(E_RANGE, "the workspace has %zu of %zu bytes", workspace_bytes, need);
    if ((int64_t)window >= (int64_t)d.max_blocks * d.page_size) window = 0;          // no key is that far back
    a.q = (const bf16*)q; a.ldq = ldq; a.out = (bf16*)out; a.ldo = ldo;
    a.k_pages = (char*)d.k_pages + layer * layer_bytes(d); a.v_pages = (char*)d.v_pages + layer * layer_bytes(d);
    a.k_scale = d.k_scale ? d.k_scale + (size_t)layer * d.kv_heads : nullptr;
    a.v_scale = d.v_scale ? d.v_scale + (size_t)layer * d.kv_heads : nullptr;
    a.table = d.block_table; a.lens = d.lens; a.seqs = seqs; a.cu = cu_tokens;
    a.window = window; a.scale = scale; a.precise = p->precise;
    a.most_keys = window && window < 0x7fffffff - a.tile_rows - 65 ? window + a.tile_rows / a.G + 65 : 0x7fffffff;
    a.part_o = (float*)workspace;
    a.part_ml = need ? a.part_o + paged_partial_floats(&a) : nullptr;
    a.info = need ? (int*)(a.part_ml + (size_t)a.target * a.kv_heads * a.tile_rows * 2) : nullptr;
    RUN("paged attention", paged_attention(&a, d.kv_type == AHA_KV_E4M3, (hipStream_t)st));
    return 0;
}
