// Block tables and slot maps of the paged key-value cache, on the device: which pages a sequence owns, and where each new token goes.
//
// reserve:  request i has c_i new tokens behind the len_i its sequence holds.  It needs ceil((len_i + c_i) / P) - ceil(len_i / P) pages; the
//           requests' needs, summed in order, say which entries of the free list they take, counted from its end.  Token t of request i
//           has position len_i + t and slot page(position / P) * P + position % P.
// truncate: the pages behind the first ceil(new_len / P) go back to the free list, in the order in which a reserve of the same requests
//           takes them: a truncate to the old lengths leaves the list as it was before the reserve, entry by entry.  A table entry that is no
//           page (attention lets callers drop the pages before a window) has nothing to give back: it is passed over, never put on the list.
//
// One workgroup does a call: the work is a prefix sum over the requests and a few words per page and token, and what bounds it is the chain
// sequence -> length -> sum -> free entry -> store, each link a trip to the L2 or memory.  All requests are looked at before anything is
// written, so a call that cannot be done (status) changes nothing.  Pages and tokens are dealt out flat, a thread finds the request of its
// page or token by bisection of the sums in LDS: a request of two thousand tokens does not keep one thread busy.  16 requests of a token: reserve
// 4.5 us, truncate 3.6; 256 of some 250 tokens (64,518): 7.6 and 4.5 for the slots, truncate 6.7.
#include "paged.h"

struct Scan2 { int a, b; };

// inclusive prefix sums of two numbers over the workgroup; totals in *all
static __device__ __forceinline__ Scan2 block_scan(Scan2 x, Scan2* wsum, Scan2* all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int a = __shfl_up(x.a, o, 64), b = __shfl_up(x.b, o, 64);
        if (lane >= o) { x.a += a; x.b += b; }
    }
    __syncthreads();                                          // wsum of an earlier scan has been read
    if (lane == 63) wsum[wave] = x;
    __syncthreads();
    Scan2 before = {0, 0}, sum = {0, 0};
    for (int w = 0; w < waves; ++w) {
        if (w == wave) before = sum;
        sum.a += wsum[w].a; sum.b += wsum[w].b;
    }
    *all = sum;
    x.a += before.a; x.b += before.b;
    return x;
}

// first i in [0, n) with end[i] > x (end is a running sum, its last value > x)
static __device__ __forceinline__ int bisect(const int* end, int n, int x) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (end[mid] > x) hi = mid; else lo = mid + 1;
    }
    return lo;
}

#define PT_THREADS 1024
// entries a thread keeps in registers from truncate's count to the list (256 requests of some 250 tokens: with a count and a list that both read them
// 11.4 us, so 6.7)
#define PT_KEEP 2
struct Request { int seq, len, count, had, need, last, err; };     // had: pages it keeps; need: pages it takes (gives back); last: its page that is filled in part

// What request i asks for; an entry with a negative sequence is padding and asks for nothing.
template <bool RESERVE>
static __device__ __forceinline__ Request look(const PagedReserveArgs& a, int i) {
    Request r = {-1, 0, 0, 0, 0, -1, 0};
    if (i >= a.n) return r;
    r.seq = a.seqs[i];
    const int c = a.counts[i];
    if (r.seq < 0) return r;
    if (r.seq >= a.t.max_seqs) { r.seq = -1; r.err = PAGED_BAD_SEQ; return r; }
    r.len = a.t.lens[r.seq];
    const int lps = a.t.lps;
    const long cap = (long)a.t.max_blocks << lps;
    if (r.len < 0 || r.len > cap) { r.err = PAGED_BAD_SEQ; return r; }
    const int P1 = (1 << lps) - 1;
    if (RESERVE) {
        if (c < 0) { r.err = PAGED_BAD_COUNT; return r; }
        if ((long)r.len + c > cap) { r.err = PAGED_TOO_LONG; return r; }
        r.count = c;
        r.had = (int)(((long)r.len + P1) >> lps);
        r.need = (int)(((long)r.len + c + P1) >> lps) - r.had;
        if (c && (r.len & P1)) {                               // new tokens go to a page that it has
            r.last = a.t.table[(long)r.seq * a.t.max_blocks + r.had - 1];
            if ((unsigned)r.last >= (unsigned)a.t.n_pages) r.err = PAGED_BAD_PAGE;
        }
    } else {
        if (c < 0 || c > r.len) { r.err = PAGED_BAD_COUNT; return r; }
        r.count = c;
        r.had = (int)(((long)c + P1) >> lps);
        r.need = (int)(((long)r.len + P1) >> lps) - r.had;
    }
    return r;
}

template <bool RESERVE>
__global__ __launch_bounds__(PT_THREADS) void paged_tables_kernel(PagedReserveArgs a, int map_tokens) {
    __shared__ unsigned seen[PAGED_MAX_SEQS / 32];
    __shared__ Scan2 wsum[PT_THREADS / 64];
    __shared__ int pend[PT_THREADS], tend[PT_THREADS], rseq[PT_THREADS], rhad[PT_THREADS], rlen[PT_THREADS], rlast[PT_THREADS];
    __shared__ int err_s, good_s, bad_at;
    __shared__ unsigned long long pages_s, tokens_s;
    const int tid = threadIdx.x, NT = blockDim.x;
    const PagedTables& t = a.t;
    const int words = (t.max_seqs + 31) >> 5;
    for (int i = tid; i < words; i += NT) seen[i] = 0;
    if (tid == 0) { err_s = 0; good_s = 0; bad_at = 0x7fffffff; pages_s = 0; tokens_s = 0; }
    const int n_free = min(max(*t.n_free, 0), t.n_pages);
    // the list's last entries, while the requests are looked at; an entry that is no page must not be handed out
    const int e0 = RESERVE && tid < n_free ? t.free_pages[n_free - 1 - tid] : 0;
    Request r0 = look<RESERVE>(a, tid);                        // kept: with at most NT requests nothing is read twice
    __syncthreads();
    if ((unsigned)e0 >= (unsigned)t.n_pages) atomicMin(&bad_at, tid);

    // ---- look at every request
    int err = 0;
    unsigned long long pages = 0, tokens = 0;
    for (int i0 = 0; i0 < a.n; i0 += NT) {
        const Request r = i0 ? look<RESERVE>(a, i0 + tid) : r0;
        err |= r.err;
        if (r.seq >= 0) {
            const unsigned bit = 1u << (r.seq & 31);
            if (atomicOr(&seen[r.seq >> 5], bit) & bit) err |= PAGED_TWICE;
        }
        pages += r.need; tokens += RESERVE ? r.count : 0;
    }
    if (err) atomicOr(&err_s, err);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) { pages += __shfl_xor(pages, o, 64); tokens += __shfl_xor(tokens, o, 64); }
    if ((tid & 63) == 0) { atomicAdd(&pages_s, pages); atomicAdd(&tokens_s, tokens); }
    __syncthreads();
    err = err_s; pages = pages_s; tokens = tokens_s;
    unsigned long long missing = 0;
    int gone = 0;                                              // truncate: pages that go back
    Scan2 all = {0, 0};
    auto is_page = [&](int page) { return (unsigned)page < (unsigned)t.n_pages; };
    auto entry = [&](int p, int m) {                           // of a chunk of requests, whose sums are in LDS: the table's entry of its p-th page
        const int i = bisect(pend, m, p);
        return t.table + (long)rseq[i] * t.max_blocks + rhad[i] + p - (i ? pend[i - 1] : 0);
    };
    int *kept[PT_KEEP], page_of[PT_KEEP];                      // truncate of at most NT requests: a thread's first entries
    if (err) {                                                 // the sums of requests that are none say nothing
    } else if (RESERVE) {
        if (pages > (unsigned long long)n_free) { err |= PAGED_NO_PAGES; missing = pages - n_free; }
        if (tokens > (unsigned long long)a.n_tokens) err |= PAGED_MANY_TOKENS;
        if (!err && pages > (unsigned long long)NT) {          // (uniform)
            for (int p = tid + NT; p < (int)pages; p += NT)
                if ((unsigned)t.free_pages[n_free - 1 - p] >= (unsigned)t.n_pages) atomicMin(&bad_at, p);
            __syncthreads();
        }
        if (!err && (unsigned long long)bad_at < pages) err |= PAGED_BAD_PAGE;
    } else if (pages > 0x7fffffffull - 4096) err |= PAGED_BAD_SEQ;          // (more than the sums below hold: no table has as many)
    else {
        // only entries that are pages go back: how many are there?
        int good = 0;                                          // of the wave, in its first lane (whose p is the least)
        for (int i0 = 0; i0 < a.n; i0 += NT) {
            const Request r = i0 ? look<RESERVE>(a, i0 + tid) : r0;
            pend[tid] = block_scan({r.need, 0}, wsum, &all).a; rseq[tid] = r.seq; rhad[tid] = r.had;
            __syncthreads();
            const int m = min(NT, a.n - i0);
#pragma unroll
            for (int k = 0; k < PT_KEEP; ++k) kept[k] = tid + k * NT < all.a ? entry(tid + k * NT, m) : nullptr;
#pragma unroll
            for (int k = 0; k < PT_KEEP; ++k) page_of[k] = kept[k] ? *kept[k] : -1;
#pragma unroll
            for (int k = 0; k < PT_KEEP; ++k) good += __popcll(__ballot(is_page(page_of[k])));
            for (int p = tid + PT_KEEP * NT; p < all.a; p += NT) good += __popcll(__ballot(is_page(*entry(p, m))));
            __syncthreads();
        }
        if ((tid & 63) == 0) atomicAdd(&good_s, good);
        __syncthreads();
        gone = good_s;
        if ((long)gone + n_free > t.n_pages) err |= PAGED_BAD_SEQ;       // more pages than the pool has: the tables are not its own
    }
    if (tid == 0) {
        a.status[0] = err;
        a.status[1] = missing > 0x7fffffffull ? 0x7fffffff : (int)missing;
    }
    if (err) {                                                 // uniform: nothing is taken, every token goes nowhere
        if (RESERVE) {
            for (int i = tid; i <= a.n; i += NT) a.cu[i] = 0;
            for (int i = tid; i < a.n_tokens; i += NT) { a.slots[i] = -1; a.positions[i] = -1; }
        }
        return;
    }

    // ---- deal out pages and tokens
    Scan2 base = {0, 0};                                       // (truncate: of entries; `back` of pages among them)
    int back = 0;
    for (int i0 = 0; i0 < a.n; i0 += NT) {
        const Request r = i0 ? look<RESERVE>(a, i0 + tid) : r0;
        if (RESERVE || a.n > NT) {                             // (else the count has left the sums as they are needed)
            const Scan2 in = block_scan({r.need, RESERVE ? r.count : 0}, wsum, &all);
            pend[tid] = in.a; tend[tid] = in.b; rseq[tid] = r.seq; rhad[tid] = r.had; rlen[tid] = r.len; rlast[tid] = r.last;
            if (RESERVE && i0 + tid < a.n) {
                a.cu[i0 + tid + 1] = base.b + in.b;
                if (i0 + tid == 0) a.cu[0] = 0;
            }
            __syncthreads();
        }
        const int m = min(NT, a.n - i0);
        if (RESERVE) {
            for (int p = tid; p < all.a; p += NT) *entry(p, m) = t.free_pages[n_free - 1 - (base.a + p)];
        } else {
            auto give = [&](int p, int* e, int page) {         // (every thread calls it)
                int at = base.a + p;                           // every entry is a page: the p-th entry is the p-th page
                if ((unsigned long long)gone != pages) {
                    Scan2 here;
                    at = back + block_scan({is_page(page), 0}, wsum, &here).a - is_page(page);
                    back += here.a;
                }
                if (is_page(page)) t.free_pages[n_free + gone - 1 - at] = page;
                if (e) *e = -1;
            };
            int p0 = 0;
            if (a.n <= NT)
#pragma unroll
                for (int k = 0; k < PT_KEEP; ++k, p0 += NT)
                    if (p0 < all.a) give(p0 + tid, kept[k], page_of[k]);
            for (; p0 < all.a; p0 += NT) {
                int* e = p0 + tid < all.a ? entry(p0 + tid, m) : nullptr;
                give(p0 + tid, e, e ? *e : -1);
            }
        }
        if (RESERVE && map_tokens)
            for (int x = tid; x < all.b; x += NT) {
                const int i = bisect(tend, m, x), off = x - (i ? tend[i - 1] : 0);
                const int pos = rlen[i] + off, blk = pos >> t.lps;
                const int page = blk < rhad[i] ? rlast[i] : t.free_pages[n_free - 1 - (base.a + (i ? pend[i - 1] : 0) + blk - rhad[i])];
                a.positions[base.b + x] = pos;
                a.slots[base.b + x] = (page << t.lps) + (pos & ((1 << t.lps) - 1));
            }
        if (r.seq >= 0) t.lens[r.seq] = RESERVE ? r.len + r.count : r.count;
        base.a += all.a; base.b += all.b;
        __syncthreads();
    }
    if (RESERVE && map_tokens)
        for (int x = base.b + tid; x < a.n_tokens; x += NT) { a.slots[x] = -1; a.positions[x] = -1; }
    if (RESERVE && a.n == 0 && tid == 0) a.cu[0] = 0;
    if (tid == 0) *t.n_free = RESERVE ? n_free - base.a : n_free + gone;
}

// The slots of many tokens, behind the tables kernel and over the whole chip: token x belongs to the request whose cu range holds it, and its
// sequence ends (now) at lens[seq].
__global__ __launch_bounds__(256) void paged_slots_kernel(PagedReserveArgs a) {
    const int x = blockIdx.x * 256 + threadIdx.x;
    if (x >= a.n_tokens) return;
    const PagedTables& t = a.t;
    if (a.status[0]) return;                                   // the tables kernel has written them
    int slot = -1, pos = -1;
    if (x < a.cu[a.n]) {
        const int i = bisect(a.cu + 1, a.n, x);
        const int seq = a.seqs[i];
        pos = t.lens[seq] - (a.cu[i + 1] - x);
        const int page = t.table[(long)seq * t.max_blocks + (pos >> t.lps)];
        if ((unsigned)page < (unsigned)t.n_pages) slot = (page << t.lps) + (pos & ((1 << t.lps) - 1));
    }
    a.slots[x] = slot;
    a.positions[x] = pos;
}

static int threads_for(int work) { return work <= 256 ? 256 : work <= 512 ? 512 : PT_THREADS; }

hipError_t paged_reserve(const PagedReserveArgs* a, hipStream_t st) {
    // Up to eight tokens a thread the tables' workgroup finds the slots too; beyond that a second launch does, over the chip.  reserve + truncate in
    // one launch against two: 16 tokens 13.6 / 16.0 us, 4,096 14.2 / 17.2, 8,192 14.0 / 16.6, 16,384 16.5 / 16.6.
    const int map = a->n_tokens <= 8 * PT_THREADS;
    const int pages = (a->n_tokens >> a->t.lps) + a->n;        // at most: the longest of the loops
    paged_tables_kernel<true><<<1, threads_for(map && a->n_tokens > pages ? a->n_tokens : pages), 0, st>>>(*a, map);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && !map) {
        paged_slots_kernel<<<(a->n_tokens + 255) / 256, 256, 0, st>>>(*a);
        e = hipGetLastError();
    }
    return e;
}
hipError_t paged_truncate(const PagedReserveArgs* a, hipStream_t st) {
    paged_tables_kernel<false><<<1, threads_for(8 * a->n), 0, st>>>(*a, 0);          // (how many pages come back is not known here: eight a request)
    return hipGetLastError();
}
