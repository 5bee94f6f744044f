// Attention of new tokens over their sequences' pages.
//
// Request i has T_i consecutive query tokens, the last of them at the last of its sequence's L_i keys: token t is at position L_i - T_i + t and
// sees the keys at and before it, the nearest `window` of them if there is one.  The G query heads of a key-value head share its keys: they
// and the tokens are the rows of one matrix product, row r = t * G + g.
//
// Structure: S^T = K Q^T and O^T += V^T P^T with v_mfma_f32_16x16x32_bf16.  A lane then holds the scores of ONE row (lane & 15) for four
// consecutive keys a tile, the softmax's maximum and sum over keys are in-register steps and two lane exchanges, and the exponentials, packed
// to bf16, are the second product's operand as they stand.  K fragments come straight from the pages (16 bytes a lane), V goes through LDS,
// where ds_read_b64_tr_b16 hands out its transpose.  The softmax runs in one pass with a running maximum and sum in fp32 (base 2).
//
// Split: a workgroup takes a tile of rows of one request, one key-value head and one chunk of the keys; chunks are joined by a second launch.
// Nothing about the lengths is known on the host, so every workgroup works out the split from them by itself (schedule()).
#include "paged.h"

typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
typedef const __attribute__((address_space(4))) int* table_t;         // read by scalar loads: nothing writes the tables while a call runs

// ---------------------------------------------------------------------------------------------
// The split.  Request i: R_i = G * T_i rows in rt_i tiles of TR, at most nb_i blocks of 64 keys a tile.  A tile is cut into C_i = ceil(nb_i / S) equal
// chunks, S being the shortest of some lengths for which sum rt_i * C_i <= target, the workgroups that run at once: no workgroup works
// longer than S, and none waits for a second round.  The lengths tried are multiples of W / target, W = sum rt_i * nb_i, at least min_blocks; where
// none is long enough (more tiles than workgroups) the last, under which there are target + (number of tiles) items at most.  Items are
// numbered request by request, tile by tile.
//   Only tiles of two chunks or more have partial results, in slots numbered the same way.  There are never more than `target` of them: either all
// items are no more, or S is at least 2.5 W / target, and C >= 2 means C <= 2 (C - 1) < 2 nb / S, so that they are fewer than 2 W / S = 0.8 target.
// The workspace therefore does not grow with the tokens (8,192 tokens, 28 / 4 heads of 128: 34 MB, with a slot for each item 154 MB).
// ---------------------------------------------------------------------------------------------
struct Work { int req, seq, q0, T, L, first, slot0, tile, chunk, chunks, slot; };

static __device__ __forceinline__ void request_shape(const PagedAttnArgs& a, int i, int* seq, int* q0, int* T, int* L) {
    *seq = a.seqs[i];
    int c0 = a.cu[i], c1 = a.cu[i + 1];
    c0 = min(max(c0, 0), a.n_tokens);
    c1 = min(max(c1, c0), a.n_tokens);
    *q0 = c0;
    if ((unsigned)*seq < (unsigned)a.max_seqs) {
        *T = c1 - c0;
        *L = min(max(a.lens[*seq], 0), a.max_blocks << a.lps);
    } else { *T = 0; *L = 0; }                              // padding: its rows are nobody's and stay as they are
}
template <int TR>
static __device__ __forceinline__ void request_tiles(const PagedAttnArgs& a, int T, int L, int* rt, int* nb) {
    *rt = (T * a.G + TR - 1) / TR;
    *nb = (min(L, a.most_keys) + 63) >> 6;
}
// (nb / S is W / S at most, so the error of a reciprocal is far below the 1e-3)
static __device__ __forceinline__ int chunks_of(const PagedAttnArgs& a, int nb, float inv_S) {
    return min(max((int)ceilf(__builtin_fmaf((float)nb, inv_S, -1e-3f)), 1), a.cmax);
}
// n / d for 0 <= n < 2^31
static __device__ __forceinline__ int quot(int n, PagedDiv d) { return (int)((__umulhi((unsigned)n, d.mul) + (unsigned)n) >> d.shift); }
// running sum over the wave's lanes (data-parallel moves: no trip through LDS); the last lane has the total
template <class T>
static __device__ __forceinline__ T wave_scan(T x) {
    static_assert(sizeof(T) == 4, "");
#define PAGED_ADD(ctrl, rows) x += __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), ctrl, rows, 0xf, false))
    PAGED_ADD(0x111, 0xf); PAGED_ADD(0x112, 0xf); PAGED_ADD(0x114, 0xf); PAGED_ADD(0x118, 0xf);       // within rows of sixteen
    PAGED_ADD(0x142, 0xa); PAGED_ADD(0x143, 0xc);                                                    // the last lane of the rows before
#undef PAGED_ADD
    return x;
}
template <class T>
static __device__ __forceinline__ T wave_total(T x) {
    return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wave_scan(x)), 63));
}
static __device__ __forceinline__ float wave_top(float x) {               // maximum, the same way
#define PAGED_MAX(ctrl, rows) x = fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, x), __builtin_bit_cast(int, x), ctrl, rows, 0xf, false)))
    PAGED_MAX(0x111, 0xf); PAGED_MAX(0x112, 0xf); PAGED_MAX(0x114, 0xf); PAGED_MAX(0x118, 0xf);
    PAGED_MAX(0x142, 0xa); PAGED_MAX(0x143, 0xc);
#undef PAGED_MAX
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}
#define TRIES 8
// what item `item` is, in scalars; false: there are fewer.  Up to 64 requests every wave looks at all of them by itself.
template <int NTH, int TR>
static __device__ __forceinline__ bool schedule(const PagedAttnArgs& a, int item, Work* out) {
    __shared__ float fsum[NTH / 64];
    __shared__ int isum[TRIES][NTH / 64];
    __shared__ Work found;
    __shared__ int have;
    const float tries[TRIES] = {1.f, 1.06f, 1.13f, 1.22f, 1.35f, 1.55f, 1.85f, 2.5f};
    const bool few = a.n <= 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, me = few ? lane : tid, step = few ? 64 : NTH;
    int seq = 0, q0 = 0, T = 0, L = 0, rt = 0, nb = 0;
    float W = 0.f;
    for (int i = me; i < a.n; i += step) {
        request_shape(a, i, &seq, &q0, &T, &L);
        request_tiles<TR>(a, T, L, &rt, &nb);
        W += (float)rt * (float)nb;
    }
    W = wave_total(W);
    if (!few) {
        if (tid == 0) have = 0;
        if (lane == 0) fsum[wave] = W;
        __syncthreads();
        W = 0.f;
#pragma unroll
        for (int k = 0; k < NTH / 64; ++k) W += fsum[k];
    }
    const float S0 = W * a.inv_target, least = (float)a.min_blocks;
    int cnt[TRIES];                                         // up to 1,023 a lane: two counts of 64 lanes in a word, and more than `target`
    float inv_S[TRIES];
#pragma unroll
    for (int k = 0; k < TRIES; ++k) { cnt[k] = 0; inv_S[k] = __builtin_amdgcn_rcpf(fmaxf(least, S0 * tries[k])); }
    for (int i = me; i < a.n; i += step) {
        if (a.n > step) { request_shape(a, i, &seq, &q0, &T, &L); request_tiles<TR>(a, T, L, &rt, &nb); }
#pragma unroll
        for (int k = 0; k < TRIES; ++k) cnt[k] = min(cnt[k] + rt * chunks_of(a, nb, inv_S[k]), 1023);
    }
#pragma unroll
    for (int k = 0; k < TRIES; k += 2) {
        const unsigned both = (unsigned)wave_total(cnt[k] | cnt[k + 1] << 16);
        cnt[k] = both & 0xffff; cnt[k + 1] = both >> 16;
    }
    if (!few) {
        if (lane == 0)
#pragma unroll
            for (int k = 0; k < TRIES; ++k) isum[k][wave] = cnt[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < TRIES; ++k) {
            cnt[k] = 0;
#pragma unroll
            for (int x = 0; x < NTH / 64; ++x) cnt[k] += isum[k][x];
        }
    }
    float S = inv_S[TRIES - 1];                             // (its reciprocal)
#pragma unroll
    for (int k = TRIES - 2; k >= 0; --k)
        if (cnt[k] <= a.target) S = inv_S[k];
    int base = 0;
    Work f;
    if (few) {
        const int C = chunks_of(a, nb, S), items = me < a.n ? rt * C : 0, cut = C > 1 ? items : 0;
        const int x = wave_scan(items), xc = wave_scan(cut);
        const int k = item - (x - items);
        const unsigned long long at = __ballot(k >= 0 && k < items);
        if (!at) return false;
        const int src = __ffsll(at) - 1;
        const int tile = (int)((unsigned)(k & 0xffffff) / (unsigned)(C & 0xffff));
        f = {src, seq, q0, T, L, item - k, xc - cut, tile, k - tile * C, C, xc - cut + k};
        out->req = src; out->seq = __builtin_amdgcn_readlane(f.seq, src); out->q0 = __builtin_amdgcn_readlane(f.q0, src);
        out->T = __builtin_amdgcn_readlane(f.T, src); out->L = __builtin_amdgcn_readlane(f.L, src); out->first = __builtin_amdgcn_readlane(f.first, src);
        out->tile = __builtin_amdgcn_readlane(f.tile, src); out->chunk = __builtin_amdgcn_readlane(f.chunk, src);
        out->chunks = __builtin_amdgcn_readlane(f.chunks, src); out->slot0 = __builtin_amdgcn_readlane(f.slot0, src); out->slot = __builtin_amdgcn_readlane(f.slot, src);
    } else {
        int base_cut = 0;
        for (int i0 = 0; i0 < a.n; i0 += NTH) {
            int C = 1, items = 0;
            if (a.n > NTH) {                                // one request a thread: its numbers are still at hand
                rt = nb = 0;
                if (i0 + tid < a.n) { request_shape(a, i0 + tid, &seq, &q0, &T, &L); request_tiles<TR>(a, T, L, &rt, &nb); }
            }
            if (i0 + tid < a.n) { C = chunks_of(a, nb, S); items = rt * C; }
            const int cut = C > 1 ? items : 0, x = wave_scan(items), xc = wave_scan(cut);
            __syncthreads();
            if (lane == 63) { isum[0][wave] = x; isum[1][wave] = xc; }
            __syncthreads();
            int before = base, before_cut = base_cut;
            for (int k = 0; k < NTH / 64; ++k) {
                if (k < wave) { before += isum[0][k]; before_cut += isum[1][k]; }
                base += isum[0][k]; base_cut += isum[1][k];
            }
            const int k = item - (before + x - items);
            if (k >= 0 && k < items) {
                found = {i0 + tid, seq, q0, T, L, item - k, before_cut + xc - cut, k / C, k % C, C, before_cut + xc - cut + k};
                have = 1;
            }
            __syncthreads();
            if (have) break;
        }
        if (!have) return false;
        f = found;
        out->req = __builtin_amdgcn_readfirstlane(f.req); out->seq = __builtin_amdgcn_readfirstlane(f.seq);
        out->q0 = __builtin_amdgcn_readfirstlane(f.q0); out->T = __builtin_amdgcn_readfirstlane(f.T); out->L = __builtin_amdgcn_readfirstlane(f.L);
        out->first = __builtin_amdgcn_readfirstlane(f.first); out->tile = __builtin_amdgcn_readfirstlane(f.tile);
        out->chunk = __builtin_amdgcn_readfirstlane(f.chunk); out->chunks = __builtin_amdgcn_readfirstlane(f.chunks);
        out->slot0 = __builtin_amdgcn_readfirstlane(f.slot0); out->slot = __builtin_amdgcn_readfirstlane(f.slot);
    }
    // for the join: where a request's partial results are
    if (item == out->first && (int)blockIdx.x == item * a.kv_heads && tid == 0 && a.cmax > 1) { a.info[2 * out->req] = out->slot0; a.info[2 * out->req + 1] = out->chunks; }
    return true;
}

// the keys [lo, hi) that any row of tile `tile` sees, as blocks of 64 from lo rounded down; chunk c of C holds blocks [c * S, min(nb, (c+1) * S))
struct Span { int lo, hi, first, nb, S; };
static __device__ __forceinline__ Span tile_span(const PagedAttnArgs& a, const Work& w, int tile, int TR) {
    Span s;
    const int t0 = quot(tile * TR, a.by_G), t1 = min(quot(tile * TR + TR - 1, a.by_G), w.T - 1);
    s.hi = max(0, min(w.L, w.L - w.T + t1 + 1));
    s.lo = a.window ? max(0, w.L - w.T + t0 + 1 - a.window) : 0;
    s.first = s.lo & ~63;
    s.nb = s.hi > s.lo ? (s.hi - s.first + 63) >> 6 : 0;
    s.S = max(1, (s.nb + w.chunks - 1) / w.chunks);
    return s;
}

// a chunk without keys says so to the join, which then leaves its partial output alone
template <int TR>
static __device__ __forceinline__ void no_keys(const PagedAttnArgs& a, int slot, int hk) {
    for (int r = threadIdx.x; r < TR; r += blockDim.x) {
        float* ml = a.part_ml + (((long)slot * a.kv_heads + hk) * TR + r) * 2;
        ml[0] = -INFINITY; ml[1] = 0.f;
    }
}
// what turns a product of q and k into an exponent of 2.  Never zero (keys of a head with scale 0, or a product of scales below the least float): hidden
// scores are -infinity before it is applied, and -infinity * 0 is no number; at the least normal number every visible score still is one of 0.
template <bool E4M3>
static __device__ __forceinline__ float log2_scale(const PagedAttnArgs& a, int hk) {
    const float c = a.scale * (E4M3 && a.k_scale ? a.k_scale[hk] : 1.f) * 1.4426950408889634f;
    return c == 0.f ? 1.17549435e-38f : c;
}
static __device__ __forceinline__ bool nonfinite(bf16x8 v) {
    const u32x4 u = __builtin_bit_cast(u32x4, v);
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) bad |= (u[i] & 0x7f800000u) == 0x7f800000u || (u[i] & 0x7f80u) == 0x7f80u;
    return bad;
}
static __device__ __forceinline__ bf16x8 e4m3x8(unsigned lo, unsigned hi) {        // exact: every e4m3 value is a bf16 value
    bf16x8 r;
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true);
    r[0] = a[0]; r[1] = a[1]; r[2] = b[0]; r[3] = b[1]; r[4] = c[0]; r[5] = c[1]; r[6] = d[0]; r[7] = d[1];
    return r;
}

#ifndef PAGED_HALVES
// ---------------------------------------------------------------------------------------------
// Few rows (one token: the G rows of a key-value head): bound by the bytes of K and V.  A workgroup's four waves take blocks of 32 keys in turn,
// each with a softmax of its own and no barrier in the loop, and are merged at the end.  The matrix cores have time to spare, so P goes into
// the product as two bf16 halves (high and remainder): no precision is lost to its rounding (2^-17 of p).  28 / 4 heads of 128: 16 tokens over
// 12,000 keys each (393 MB) 72 us, 5.4 TB/s; 64 over 9,000 in e4m3 (590 MB) 109 us, 5.4 TB/s (a large copy: 4.9).  One over 2,048 keys 7.2 us: the
// chain of request, length, table, keys, merge, each link a trip to memory.
// ---------------------------------------------------------------------------------------------
template <int D, bool E4M3>
__global__ __launch_bounds__(256) void paged_attn_rows_kernel(PagedAttnArgs a) {
    constexpr int KSQ = D / 32, DT = D / 16, VST = D + 16, TR = 16;
    constexpr int NK = E4M3 ? KSQ / 2 : KSQ;               // 16-byte loads of one K tile a lane
    constexpr int NV = E4M3 ? D / 32 : D / 16;             // 16-byte loads of 32 V rows a lane
    constexpr int VCH = E4M3 ? D / 16 : D / 8;             // 16-byte chunks of a V row
    __shared__ __attribute__((aligned(16))) bf16 Vs[4][32 * VST];
    __shared__ float sm[4][16], sl[4][16];

    const int item = quot(blockIdx.x, a.by_kv_heads), hk = blockIdx.x - item * a.kv_heads;
    Work w;
    if (!schedule<256, TR>(a, item, &w)) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int q4 = lane >> 4, r16 = lane & 15;
    const Span sp = tile_span(a, w, w.tile, TR);
    const int b0 = w.chunk * sp.S, b1 = min(sp.nb, b0 + sp.S);
    if (b0 >= b1 && w.chunks > 1) { no_keys<TR>(a, w.slot, hk); return; }
    const int R = w.T * a.G, base_pos = w.L - w.T;

    // this lane's row and its query
    bf16x8 qf[KSQ];
    const int my_r = min(w.tile * TR + r16, R - 1), my_t = quot(my_r, a.by_G), pos = base_pos + my_t;
    {
        const bf16* qp = a.q + (long)(w.q0 + my_t) * a.ldq + (long)(hk * a.G + my_r - my_t * a.G) * a.hd;
        const bf16x8 z8 = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int ks = 0; ks < KSQ; ++ks) {
            // E4M3: a lane's 16 bytes of a K row are 16 channels, the operands of two products; the queries follow that order
            const int ch = E4M3 ? (ks >> 1) * 64 + q4 * 16 + (ks & 1) * 8 : ks * 32 + q4 * 8;
            const bf16x8 v = *(const bf16x8*)(qp + min(ch, a.hd - 8));
            qf[ks] = ch < a.hd ? v : z8;
        }
    }
    const int pos_min = base_pos + quot(w.tile * TR, a.by_G), pos_max = base_pos + min(quot(w.tile * TR + TR - 1, a.by_G), w.T - 1);
    const bool one_pos = pos_min == pos_max;
    const float c2 = log2_scale<E4M3>(a, hk);

    f32x4 o[DT];
    float m_run = -INFINITY, l_run = 0.f;
#pragma unroll
    for (int i = 0; i < DT; ++i) o[i] = (f32x4){0.f, 0.f, 0.f, 0.f};

    constexpr int ES = E4M3 ? 1 : 2;
    const long head_bytes = ((long)a.hd << a.lps) * ES;     // one head of one page
    const char* kp = (const char*)a.k_pages + hk * head_bytes;
    const char* vp = (const char*)a.v_pages + hk * head_bytes;
    const long page_bytes = head_bytes * a.kv_heads;
    const table_t table = (table_t)(uintptr_t)(a.table + (long)w.seq * a.max_blocks);
    const int P1 = (1 << a.lps) - 1;
    u32x4 kreg[2][NK], vreg[NV];
    bool page_ok[2];
    // a block's two tiles of sixteen keys: their pages (an entry that is no page is read as page 0 and masked)
    auto tile_off = [&](int key0, bool* ok) -> long {
        const int blk = min(key0 >> a.lps, a.max_blocks - 1);
        const int page = table[blk];
        *ok = (unsigned)page < (unsigned)a.n_pages;
        return (*ok ? page : 0) * page_bytes + (long)(key0 & P1) * a.hd * ES;
    };
    long off[2];
    auto load_v = [&]() {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int idx = i * 64 + lane, row = idx / VCH, ch = idx % VCH;
            const long ro = (row < 16 ? off[0] : off[1]) + (long)(row & 15) * a.hd * ES;
            vreg[i] = *(const u32x4*)(vp + ro + min(ch * 16, a.hd * ES - 16));
        }
    };
    auto load_k = [&]() {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int i = 0; i < NK; ++i) {
                const int cb = (i * 4 + q4) * 16;           // byte of the row
                kreg[kt][i] = *(const u32x4*)(kp + off[kt] + (long)r16 * a.hd * ES + min(cb, a.hd * ES - 16));
            }
    };
    bf16* vs = Vs[wave];
    const int k_end = min(sp.hi, sp.first + b1 * 64);
    int key0 = sp.first + b0 * 64 + wave * 32;
    if (key0 < k_end) {
        off[0] = tile_off(key0, &page_ok[0]); off[1] = tile_off(key0 + 16, &page_ok[1]);
        load_v(); load_k();
    }
    for (; key0 < k_end; key0 += 128) {
        const bool ok0 = page_ok[0], ok1 = page_ok[1];
        const bool plain = ok0 && ok1 && key0 + 31 <= pos_min && key0 + 31 < k_end && (!a.window || key0 > pos_max - a.window);
        // ---- V to LDS; rows that no row of the tile sees become zero (their bytes may be anything)
        bool odd = false;                                   // a value that is not finite in a row that some see and others do not
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int idx = i * 64 + lane, row = idx / VCH, ch = idx % VCH;
            bf16x8 v0, v1;
            if constexpr (E4M3) { v0 = e4m3x8(vreg[i][0], vreg[i][1]); v1 = e4m3x8(vreg[i][2], vreg[i][3]); }
            else v0 = __builtin_bit_cast(bf16x8, vreg[i]);
            const bool pad = ch * 16 >= a.hd * ES;
            bool none = pad;
            if (!plain) {
                const int j = key0 + row;
                none |= j >= k_end || j < sp.lo || !(row < 16 ? ok0 : ok1);
                if (!none && !one_pos) { odd |= nonfinite(v0); if constexpr (E4M3) odd |= nonfinite(v1); }
            }
            const bf16x8 z8 = {0, 0, 0, 0, 0, 0, 0, 0};
            if constexpr (E4M3) {
                *(bf16x8*)&vs[row * VST + ch * 16] = none ? z8 : v0;
                *(bf16x8*)&vs[row * VST + ch * 16 + 8] = none ? z8 : v1;
            } else *(bf16x8*)&vs[row * VST + ch * 8] = none ? z8 : v0;
        }
        asm volatile("" ::: "memory");
        const int kn = key0 + 128;
        if (kn < k_end) {
            off[0] = tile_off(kn, &page_ok[0]); off[1] = tile_off(kn + 16, &page_ok[1]);
            load_v();
        }
        // ---- scores: s[kt][e] is row r16's with key key0 + 16 kt + 4 q4 + e
        f32x4 s[2];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            s[kt] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < NK; ++i) {
                bf16x8 k0, k1;
                if constexpr (E4M3) { k0 = e4m3x8(kreg[kt][i][0], kreg[kt][i][1]); k1 = e4m3x8(kreg[kt][i][2], kreg[kt][i][3]); }
                else k0 = __builtin_bit_cast(bf16x8, kreg[kt][i]);
                if (a.hd < D) {                             // channels past the head: whatever was read there
                    const bf16x8 z8 = {0, 0, 0, 0, 0, 0, 0, 0};
                    if ((i * 4 + q4) * 16 >= a.hd * ES) { k0 = z8; if constexpr (E4M3) k1 = z8; }
                }
                if constexpr (E4M3) {
                    s[kt] = mfma16(k0, qf[2 * i], s[kt]);
                    s[kt] = mfma16(k1, qf[2 * i + 1], s[kt]);
                } else s[kt] = mfma16(k0, qf[i], s[kt]);
            }
        }
        if (kn < k_end) load_k();
        const bool any_odd = !plain && !one_pos && __any(odd);
        if (!plain) {
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int j = key0 + kt * 16 + 4 * q4 + e;
                    const bool see = j <= pos && j < k_end && (kt ? ok1 : ok0) && (!a.window || j > pos - a.window);
                    s[kt][e] = see ? s[kt][e] : -INFINITY;
                }
        }
        float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float m_new = fmaxf(m_run, mx * c2);
        const float ref = m_new == -INFINITY ? 0.f : m_new;                // a row that has seen nothing yet: 2^(-inf) = 0 throughout
        const float alpha = __builtin_amdgcn_exp2f(m_run - ref);
        float psum = 0.f;
        bf16x8 ph, pl;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][e], c2, -ref));
                psum += p;
                const bf16 hi = f2bf(p);
                ph[kt * 4 + e] = hi;
                pl[kt * 4 + e] = f2bf(p - bf2f(hi));
            }
        m_run = m_new;
        l_run = l_run * alpha + psum;
#pragma unroll
        for (int i = 0; i < DT; ++i) o[i] *= alpha;
        // ---- O^T += V^T P^T: slot (q4, e) is key 4 q4 + e of the first tile, of the second from e = 4
        const int vrow = 4 * q4 + (r16 >> 2), vcol = 4 * (r16 & 3);
        auto v_frag = [&](int dt) {
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(&vs[vrow * VST + dt * 16 + vcol]));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(&vs[(16 + vrow) * VST + dt * 16 + vcol]));
            return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        };
        if (!any_odd) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const bf16x8 vf = v_frag(dt);
                o[dt] = mfma16(vf, ph, o[dt]);
                o[dt] = mfma16(vf, pl, o[dt]);
            }
        } else {
            // 0 * inf would carry a value into rows that do not see its key: each position's rows on their own, with the keys they see
            for (int p = pos_min; p <= pos_max; ++p) {
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    bf16x8 vf = v_frag(dt);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int j = key0 + (e >> 2) * 16 + 4 * q4 + (e & 3);
                        if (j > p || (a.window && j <= p - a.window)) vf[e] = 0;
                    }
                    f32x4 t = mfma16(vf, ph, o[dt]);
                    t = mfma16(vf, pl, t);
                    o[dt] = pos == p ? t : o[dt];
                }
            }
        }
        asm volatile("" ::: "memory");
    }

    // ---- merge the four waves: O of the sixteen rows in LDS
    constexpr int OST = D + 4, E = D / 16;
    static_assert(4 * 16 * OST * 4 <= (int)sizeof(Vs), "the merge uses V's LDS");
    float* ob = (float*)&Vs[0][0];
    l_run += __shfl_xor(l_run, 16, 64);
    l_run += __shfl_xor(l_run, 32, 64);
    __syncthreads();
    if (q4 == 0) { sm[wave][r16] = m_run; sl[wave][r16] = l_run; }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) *(f32x4*)&ob[(wave * 16 + r16) * OST + dt * 16 + 4 * q4] = o[dt];
    __syncthreads();
    const int row = tid >> 4, c = (tid & 15) * E, r = w.tile * TR + row;
    const float M = fmaxf(fmaxf(sm[0][row], sm[1][row]), fmaxf(sm[2][row], sm[3][row])), ref = M == -INFINITY ? 0.f : M;
    float acc[E], lsum = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        const float f = __builtin_amdgcn_exp2f(sm[x][row] - ref);
        lsum += sl[x][row] * f;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += ob[(x * 16 + row) * OST + c + e] * f;
    }
    if (r >= R) return;
    if (w.chunks == 1) {
        // a row that sees no key is zero; NaN stays
        const float inv = lsum > 0.f ? (E4M3 && a.v_scale ? a.v_scale[hk] : 1.f) / lsum : lsum == 0.f ? 0.f : lsum;
        const int t = quot(r, a.by_G);
        bf16* op = a.out + (long)(w.q0 + t) * a.ldo + (long)(hk * a.G + r - t * a.G) * a.hd;
#pragma unroll
        for (int e = 0; e < E; ++e) if (c + e < a.hd) op[c + e] = f2bf(acc[e] * inv);
    } else {
        const long pr = ((long)w.slot * a.kv_heads + hk) * TR + row;
#pragma unroll
        for (int e = 0; e < E; ++e) a.part_o[pr * D + c + e] = acc[e];
        if (c == 0) { a.part_ml[pr * 2] = M; a.part_ml[pr * 2 + 1] = lsum; }
    }
}

#endif
// ---------------------------------------------------------------------------------------------
// Many rows (frames, prompts): bound by the matrix cores and the exponentials.  A workgroup's four waves have 16 NT rows each and share blocks of
// 64 keys, K and V double-buffered in LDS, with one barrier a block.  bf16 pages go straight to LDS (buffer_load ... lds, 1 KiB of contiguous rows an
// instruction), e4m3 through registers, where they become bf16.  The next block is under way during the first product and the softmax; bf16: the second
// product begins with a wait for it, as the compiler cannot tell its transposing reads of V from the transfers into the other buffer.  In LDS a row's
// 16-byte chunks are permuted by its number: sixteen rows read at one column, or eight rows at two, touch every bank once.
// P is rounded to bf16 (half a step, 2^-8 of p, as the output itself is) unless the caller asks for two halves (HALVES: 2^-17); the sum of the row is
// taken from the rounded values, by the matrix cores (a product with ones), so that numerator and denominator round alike.  One half / two, us: 8,192
// tokens over as many keys 487 / 703, 8 x 36 over 12,000 78 / 101, 16 x 5 over 5,000 39.8 / 40.4, x 7 in e4m3 30.5 / 34.8.  The running maximum moves only when a score exceeds it by 2^8: until
// then the exponentials stay below 2^8 and neither the sum nor the output is rescaled.  28 / 4 heads of 128: 8,192 tokens over as many keys 481 us,
// 1,000 TFLOP/s of the pairs a row sees (a large library product: 1,430), 8 / 2 heads of 64 562; 4 x 2,048 over 8,192 keys 848 us,
// of which 800 stay without the exponentials, 751 without staging, 738 without the second product: none of them alone bounds it.  8 x 36 tokens
// over 12,000 keys 70 us, about 15 of them the start and 33 MB of partial results.
// ---------------------------------------------------------------------------------------------
template <int D> struct TileLds {
    static constexpr int CPR = D / 8, RPP = 64 / CPR;       // 16-byte chunks of a row; rows of a 1-KiB piece
    static __device__ __forceinline__ int k_slot(int row, int ch) { return row * D + ((ch ^ (D == 128 ? row & 15 : (row >> 1) & 7)) << 3); }
    static __device__ __forceinline__ int v_slot(int row, int ch) { return row * D + ((ch ^ (D == 128 ? 2 * (row & 7) : 2 * ((row >> 1) & 3))) << 3); }
};
// sixteen bytes a lane, from its offset in `from` to lane * 16 behind `lds`
static __device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t from, bf16* lds, unsigned off) {
#ifdef __HIP_DEVICE_COMPILE__
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void*)lds, 16, off, 0, 0, 0);
#endif
}

template <int D, bool E4M3, int NT, bool HALVES>
__global__ __launch_bounds__(256, 2) void paged_attn_tile_kernel(PagedAttnArgs a) {
    constexpr int KSQ = D / 32, DT = D / 16, TR = 64 * NT, BLK = 64 * D;
    using LD = TileLds<D>;
    extern __shared__ __attribute__((aligned(16))) bf16 kv[];             // [buffer][K, V][64][D]
    __shared__ int odd_s[2];

    const int item = quot(blockIdx.x, a.by_kv_heads), hk = blockIdx.x - item * a.kv_heads;
    Work w;
    if (!schedule<256, TR>(a, item, &w)) return;
    w.tile = (w.T * a.G + TR - 1) / TR - 1 - w.tile;         // the longest rows of a prompt first
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int q4 = lane >> 4, r16 = lane & 15;
    const Span sp = tile_span(a, w, w.tile, TR);
    const int b0 = w.chunk * sp.S, b1 = min(sp.nb, b0 + sp.S);
    if (b0 >= b1 && w.chunks > 1) { no_keys<TR>(a, w.slot, hk); return; }
    const int R = w.T * a.G, base_pos = w.L - w.T;
    const int row0 = w.tile * TR + wave * 16 * NT;
    const bool wave_on = row0 < R;

    int pos[NT];
    bf16x8 qf[NT][KSQ];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int r = min(row0 + nt * 16 + r16, R - 1), t = quot(r, a.by_G), g = r - t * a.G;
        pos[nt] = base_pos + t;
        const bf16* qp = a.q + (long)(w.q0 + t) * a.ldq + (long)(hk * a.G + g) * a.hd;
        const bf16x8 z8 = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int ks = 0; ks < KSQ; ++ks) {
            const int ch = ks * 32 + q4 * 8;
            const bf16x8 v = *(const bf16x8*)(qp + min(ch, a.hd - 8));
            qf[nt][ks] = ch < a.hd ? v : z8;
        }
    }
    // the positions of the workgroup's rows, and of the wave's
    const int pos_lo = base_pos + quot(w.tile * TR, a.by_G), pos_hi = base_pos + min(quot(w.tile * TR + TR - 1, a.by_G), w.T - 1);
    const int wpos_lo = base_pos + quot(min(row0, R - 1), a.by_G), wpos_hi = base_pos + quot(min(row0 + 16 * NT - 1, R - 1), a.by_G);
    const float c2 = log2_scale<E4M3>(a, hk);

    f32x4 o[NT][DT], lacc[NT];
    float m_run[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        m_run[nt] = -INFINITY; lacc[nt] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < DT; ++i) o[nt][i] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }

    constexpr int ES = E4M3 ? 1 : 2;
    const int row_bytes = a.hd * ES;
    const long head_bytes = ((long)a.hd << a.lps) * ES, page_bytes = head_bytes * a.kv_heads;
    const char* kp = (const char*)a.k_pages + hk * head_bytes;
    const char* vp = (const char*)a.v_pages + hk * head_bytes;
    const table_t table = (table_t)(uintptr_t)(a.table + (long)w.seq * a.max_blocks);
    const int P1 = (1 << a.lps) - 1;
    // the pages of a block's four tiles of sixteen keys (scalar loads; an entry that is no page is read as page 0 and masked); looked up two
    // blocks ahead
    auto look_up = [&](int key0, int i) { return table[min((key0 + 16 * i) >> a.lps, a.max_blocks - 1)]; };
    auto no_page = [&](int page) { return (unsigned)page >= (unsigned)a.n_pages; };
    constexpr int NL = E4M3 ? D / 64 : D / 32;              // 16-byte loads a lane of sixteen rows
    u32x4 kreg[NL], vreg[NL];
    // a lane's byte offsets within sixteen rows: in LDS a row's chunk c lies in place c ^ f(row), so the lane of that place asks for it; chunks
    // past the head lie behind the buffer, where a load is zero (a copy of the row's own values could be infinite, and 0 * inf is no zero)
    auto in_row = [&](int row, int byte) { return byte < row_bytes ? (unsigned)(row * row_bytes + byte) : 0x40000000u; };
    unsigned koff[NL], voff[NL];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        if constexpr (!E4M3) {
            const int row = i * LD::RPP + lane / LD::CPR, c = lane % LD::CPR;
            koff[i] = in_row(row, (LD::k_slot(row, c) - row * D) * 2);
            voff[i] = in_row(row, (LD::v_slot(row, c) - row * D) * 2);
        } else {
            const int idx = i * 64 + lane;
            koff[i] = voff[i] = in_row(idx / (D / 16), idx % (D / 16) * 16);
        }
    }
    auto stage = [&](int key0, int page, int buf) {         // wave w has keys 16 w .. 16 w + 15 of a block; bf16: into LDS; e4m3: into registers
        const long off = (no_page(page) ? 0 : page) * page_bytes + (long)((key0 + wave * 16) & P1) * row_bytes;
        const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc((void*)(kp + off), 0, 16 * row_bytes, 0x00020000);
        const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc((void*)(vp + off), 0, 16 * row_bytes, 0x00020000);
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            if constexpr (!E4M3) {
                load_to_lds(kr, kv + buf * 2 * BLK + (wave * 16 + i * LD::RPP) * D, koff[i]);
                load_to_lds(vr, kv + buf * 2 * BLK + BLK + (wave * 16 + i * LD::RPP) * D, voff[i]);
            } else {
                kreg[i] = __builtin_amdgcn_raw_buffer_load_b128(kr, koff[i], 0, 0);
                vreg[i] = __builtin_amdgcn_raw_buffer_load_b128(vr, voff[i], 0, 0);
            }
        }
    };
    auto unstage = [&](int buf) {                           // e4m3: from registers into LDS, as bf16
        if constexpr (E4M3) {
            constexpr int C = D / 16;
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                const int idx = i * 64 + lane, row = wave * 16 + idx / C, c = idx % C * 2;
                *(bf16x8*)(kv + buf * 2 * BLK + LD::k_slot(row, c)) = e4m3x8(kreg[i][0], kreg[i][1]);
                *(bf16x8*)(kv + buf * 2 * BLK + LD::k_slot(row, c + 1)) = e4m3x8(kreg[i][2], kreg[i][3]);
                *(bf16x8*)(kv + buf * 2 * BLK + BLK + LD::v_slot(row, c)) = e4m3x8(vreg[i][0], vreg[i][1]);
                *(bf16x8*)(kv + buf * 2 * BLK + BLK + LD::v_slot(row, c + 1)) = e4m3x8(vreg[i][2], vreg[i][3]);
            }
        }
    };
    const bf16 one = (bf16)1.0f;
    const bf16x8 ones = {one, one, one, one, one, one, one, one};

    int buf = 0;
    // the wave's own page a block ahead; all four of the block itself, for the mask
    const bool one_page = a.lps >= 6;                       // a block lies in one page
    int mine = look_up(sp.first + b0 * 64, wave);
    int p0, p1 = 0, p2 = 0, p3 = 0;
    auto look_up_all = [&](int key0) {
        p0 = look_up(key0, 0);
        if (!one_page) { p1 = look_up(key0, 1); p2 = look_up(key0, 2); p3 = look_up(key0, 3); }
    };
    look_up_all(sp.first + b0 * 64);
    if (b0 < b1) { stage(sp.first + b0 * 64, mine, 0); unstage(0); }
    mine = look_up(sp.first + b0 * 64 + 64, wave);
    for (int b = b0; b < b1; ++b, buf ^= 1) {
        const int key0 = sp.first + b * 64;
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();                       // this block is in LDS, the other buffer is free
        unsigned bad = 0;
        if (no_page(p0) || no_page(p1) || no_page(p2) || no_page(p3))
            bad = one_page ? 15 : (no_page(p0) ? 1u : 0u) | (no_page(p1) ? 2u : 0u) | (no_page(p2) ? 4u : 0u) | (no_page(p3) ? 8u : 0u);
        const bool plain = !bad && key0 + 63 <= pos_lo && (!a.window || key0 > pos_hi - a.window);             // every row sees every key
        bool odd = false;
        if (!plain) {
            // values that no row of the workgroup sees become zero; is one that some see and others do not not finite?
            if (tid == 0) odd_s[buf] = 0;
            __syncthreads();
            bool mine_odd = false;
            for (int x = tid; x < 64 * LD::CPR; x += 256) {
                const int row = x / LD::CPR, j = key0 + row;
                bf16x8* vv = (bf16x8*)(kv + buf * 2 * BLK + BLK + x * 8);
                if (j >= sp.hi || j < sp.lo || (bad >> (row >> 4) & 1)) *vv = (bf16x8){0, 0, 0, 0, 0, 0, 0, 0};
                else mine_odd |= nonfinite(*vv);
            }
            if (mine_odd) odd_s[buf] = 1;
            __syncthreads();
            odd = odd_s[buf] != 0 && pos_lo != pos_hi;
        }
        if (b + 1 < b1) {
            stage(key0 + 64, mine, buf ^ 1);
            mine = look_up(key0 + 128, wave);
            look_up_all(key0 + 64);
        }
        // a wave whose rows see nothing of the block, or that has none, only keeps the barriers
        if (wave_on && key0 <= wpos_hi && (!a.window || key0 + 63 > wpos_lo - a.window)) {
            const bf16* ks_ = kv + buf * 2 * BLK;
            const bf16* vs_ = ks_ + BLK;
            f32x4 s[NT][4];
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) s[nt][kt] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < KSQ; ++ks) {
                    const bf16x8 kf = *(const bf16x8*)&ks_[LD::k_slot(kt * 16 + r16, ks * 4 + q4)];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) s[nt][kt] = mfma16(kf, qf[nt][ks], s[nt][kt]);
                }
            }
            __builtin_amdgcn_sched_group_barrier(0x100, 2 * KSQ, 0);      // K fragments a key tile ahead of their products
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
                __builtin_amdgcn_sched_group_barrier(0x8, NT * KSQ, 0);
                if (kt < 2) __builtin_amdgcn_sched_group_barrier(0x100, KSQ, 0);
            }
            __builtin_amdgcn_s_setprio(0);
            if (!plain && (bad || key0 + 63 > wpos_lo || (a.window && key0 <= wpos_hi - a.window))) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    int ahead = pos[nt] - key0 - 4 * q4;    // the last key the row sees, from this lane's first
                    asm volatile("" : "+v"(ahead));         // (computed here, not kept in registers through the loop)
                    const int least = a.window ? ahead - a.window : -0x40000000;
#pragma unroll
                    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const bool see = kt * 16 + e <= ahead && kt * 16 + e > least && !(bad >> kt & 1);
                            s[nt][kt][e] = see ? s[nt][kt][e] : -INFINITY;
                        }
                }
            }
            bf16x8 pb[NT][2], pr[HALVES ? NT : 1][2];           // P, and what its rounding left
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                // exponentials against the running reference; only where one of them exceeds 2^8, or a row has no reference yet, is the
                // row's maximum looked for
                float p[4][4], top = 0.f;
                auto exps = [&]() {
                    const float ref = m_run[nt] == -INFINITY ? 0.f : -m_run[nt];
                    top = 0.f;
#pragma unroll
                    for (int kt = 0; kt < 4; ++kt) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) p[kt][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[nt][kt][e], c2, ref));
                        top = fmaxf(fmaxf(top, p[kt][0]), fmaxf(p[kt][1], fmaxf(p[kt][2], p[kt][3])));
                    }
                };
                exps();
                if (__any(top > 256.f || m_run[nt] == -INFINITY)) {
                    float mx = -INFINITY;
#pragma unroll
                    for (int kt = 0; kt < 4; ++kt) mx = fmaxf(mx, fmaxf(fmaxf(s[nt][kt][0], s[nt][kt][1]), fmaxf(s[nt][kt][2], s[nt][kt][3])));
                    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
                    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
                    mx *= c2;
                    const float m_new = mx > m_run[nt] + 8.f ? mx : m_run[nt];        // (-inf + 8 = -inf: the first key a row sees)
                    const float alpha = m_new == m_run[nt] ? 1.f : __builtin_amdgcn_exp2f(m_run[nt] - m_new);
                    m_run[nt] = m_new;
#pragma unroll
                    for (int e = 0; e < 4; ++e) lacc[nt][e] *= alpha;
#pragma unroll
                    for (int i = 0; i < DT; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[nt][i][e] *= alpha;
                    exps();
                }
#pragma unroll
                for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const bf16 hi = f2bf(p[kt][e]);
                        pb[nt][kt >> 1][(kt & 1) * 4 + e] = hi;
                        if constexpr (HALVES) pr[nt][kt >> 1][(kt & 1) * 4 + e] = f2bf(p[kt][e] - bf2f(hi));
                    }
#pragma unroll
                for (int kp_ = 0; kp_ < 2; ++kp_) {
                    lacc[nt] = mfma16(ones, pb[nt][kp_], lacc[nt]);
                    if constexpr (HALVES) lacc[nt] = mfma16(ones, pr[nt][kp_], lacc[nt]);
                }
            }
            // O^T += V^T P^T: slot (q4, e) of a pair of key tiles is key 4 q4 + e of the first, of the second from e = 4
            const int vrow = 4 * q4 + (r16 >> 2), vch = (r16 & 3) >> 1, vin = 4 * (r16 & 1);
            auto v_frag = [&](int dt, int kp_) {
                const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(vs_ + LD::v_slot(kp_ * 32 + vrow, dt * 2 + vch) + vin));
                const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(vs_ + LD::v_slot(kp_ * 32 + 16 + vrow, dt * 2 + vch) + vin));
                return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
            };
            __builtin_amdgcn_s_setprio(1);
            if (!odd) {
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int kp_ = 0; kp_ < 2; ++kp_) {
                        const bf16x8 vf = v_frag(dt, kp_);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) o[nt][dt] = mfma16(vf, pb[nt][kp_], o[nt][dt]);
                        if constexpr (HALVES)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) o[nt][dt] = mfma16(vf, pr[nt][kp_], o[nt][dt]);
                    }
                if constexpr (!E4M3) {                      // (the registers of an e4m3 block under way leave no room)
                    __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);    // V fragments two channel tiles ahead
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) {
                        __builtin_amdgcn_sched_group_barrier(0x8, (HALVES ? 4 : 2) * NT, 0);
                        if (dt + 2 < DT) __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
                    }
                }
            } else {
                for (int p = wpos_lo; p <= wpos_hi; ++p) {  // each position's rows on their own, with the keys they see (0 * inf is no zero)
                    int ahead = p - key0 - 4 * q4;
                    asm volatile("" : "+v"(ahead));
                    const int least = a.window ? ahead - a.window : -0x40000000;
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                        for (int kp_ = 0; kp_ < 2; ++kp_) {
                            bf16x8 vf = v_frag(dt, kp_);
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const int j = kp_ * 32 + (e >> 2) * 16 + (e & 3);
                                if (j > ahead || j <= least) vf[e] = 0;
                            }
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                f32x4 x = mfma16(vf, pb[nt][kp_], o[nt][dt]);
                                if constexpr (HALVES) x = mfma16(vf, pr[nt][kp_], x);
                                o[nt][dt] = pos[nt] == p ? x : o[nt][dt];
                            }
                        }
                }
            }
        }
        __builtin_amdgcn_s_setprio(0);
        if (b + 1 < b1) unstage(buf ^ 1);
    }
    if (!wave_on) return;

    const float vsc = E4M3 && a.v_scale ? a.v_scale[hk] : 1.f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int r = row0 + nt * 16 + r16;
        if (r >= R) continue;
        const float l = lacc[nt][0];
        if (w.chunks == 1) {
            const float inv = l > 0.f ? vsc / l : l == 0.f ? 0.f : l;
            const int t = quot(r, a.by_G), g = r - t * a.G;
            bf16* op = a.out + (long)(w.q0 + t) * a.ldo + (long)(hk * a.G + g) * a.hd + 4 * q4;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
                if (dt * 16 < a.hd) *(bf16x4*)(op + dt * 16) = (bf16x4){f2bf(o[nt][dt][0] * inv), f2bf(o[nt][dt][1] * inv), f2bf(o[nt][dt][2] * inv), f2bf(o[nt][dt][3] * inv)};
        } else {
            const long pr = ((long)w.slot * a.kv_heads + hk) * TR + (wave * NT + nt) * 16 + r16;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) *(f32x4*)&a.part_o[pr * D + dt * 16 + 4 * q4] = o[nt][dt];
            if (q4 == 0) { a.part_ml[pr * 2] = m_run[nt]; a.part_ml[pr * 2 + 1] = l; }
        }
    }
}

template <int D, bool E4M3, int TR, bool HALVES>
static void launch_tiles(const PagedAttnArgs* a, hipStream_t st) {
    paged_attn_tile_kernel<D, E4M3, TR / 64, HALVES><<<a->grid_items * a->kv_heads, 256, 4 * 64 * D * sizeof(bf16), st>>>(*a);
}
#ifdef PAGED_HALVES                                             // (a source of its own, built beside this one: paged_attention_halves.hip)
template <int D, bool E4M3>
static void launch_halves(const PagedAttnArgs* a, hipStream_t st) {
    if (a->tile_rows == 64) launch_tiles<D, E4M3, 64, true>(a, st);
    else launch_tiles<D, E4M3, 128, true>(a, st);
}
void paged_tiles_halves(const PagedAttnArgs* a, int e4m3, hipStream_t st) {
    if (a->hd <= 64) e4m3 ? launch_halves<64, true>(a, st) : launch_halves<64, false>(a, st);
    else e4m3 ? launch_halves<128, true>(a, st) : launch_halves<128, false>(a, st);
}
#else
// ---------------------------------------------------------------------------------------------
// Joins the chunks of split rows: a wave for each token (of many tokens most have nothing to join), for each token and query head, or, where that
// leaves the chip empty, four waves for each token and head, which share its chunks.  A lane knows one chunk's maximum and sum, so the weights of
// 64 chunks take one load; then 64 / (D / 4) partial rows are added at a time.  What bounds it is the chain request -> slot -> output: the request
// is found by counting, not by bisection, and the first rows are asked for along with their weights.  56 registers let a CU hold the 32 waves of
// 8 x 36 tokens at once.  28 heads of 128: 288 tokens of 8 chunks (36 MB) 9.4 us, 16 of up to 14 chunks 5.2 us, one of 16 3.9 us.
// ---------------------------------------------------------------------------------------------
template <int D, int TR, int WAVES>
__global__ __launch_bounds__(256) void paged_attn_join_kernel(PagedAttnArgs a, int e4m3, int heads_each) {
    constexpr int LPR = D / 4, AT = 64 / LPR, FLY = WAVES == 4 ? 8 : 4;   // lanes of a row, rows at a time, loads under way
    __shared__ float sh_m[4], sh_l[4];
    __shared__ f32x4 sh_o[4][LPR];
    const int heads = a.kv_heads * a.G, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int unit = WAVES == 4 ? blockIdx.x : blockIdx.x * 4 + wave, lane = threadIdx.x & 63;
    const int tok = heads_each == 1 ? quot(unit, a.by_heads) : unit, h0 = heads_each == 1 ? unit - tok * heads : 0;    // (one head or all)
    if (tok >= a.n_tokens) return;
    int req = 0;
    if (a.n <= 512) {
        for (int i0 = 0; i0 < a.n; i0 += 64) req += __popcll(__ballot(i0 + lane < a.n && a.cu[min(i0 + lane, a.n - 1) + 1] <= tok));
    } else {
        int hi = a.n;
        while (req < hi) { const int mid = (req + hi) >> 1; if (a.cu[mid + 1] <= tok) req = mid + 1; else hi = mid; }
    }
    if (req >= a.n) return;                                 // behind the last request
    const int q0 = min(max(a.cu[req], 0), a.n_tokens), T = min(max(a.cu[req + 1], q0), a.n_tokens) - q0, seq = a.seqs[req], first = a.info[2 * req], chunks = a.info[2 * req + 1];
    if (tok < q0 || (unsigned)seq >= (unsigned)a.max_seqs || chunks <= 1) return;
    const int rt = (T * a.G + TR - 1) / TR, col = lane % LPR * 4, sub = lane / LPR;
    const int each = (chunks + WAVES - 1) / WAVES, c_lo = WAVES == 4 ? wave * each : 0, c_hi = min(chunks, c_lo + each);
    for (int h = h0; h < h0 + heads_each; ++h) {
        const int hk = quot(h, a.by_G), r = (tok - q0) * a.G + h - hk * a.G, tile = r / TR;
        const long slot = first + (long)(TR > 16 ? rt - 1 - tile : tile) * chunks;         // (the tile kernel takes a request's tiles from the last)
        if (slot < 0 || slot + chunks > a.target) return;             // (a cu that is no running sum)
        const long step = (long)a.kv_heads * TR, p0 = (slot * a.kv_heads + hk) * TR + (r - tile * TR);
        float M = -INFINITY, l = 0.f;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f}, v[FLY];
        const unsigned hop = (unsigned)step * (D * 4);      // (bytes: all partial results of a call are 67 MB at most: 1,024 x 128 rows of 512)
        const __amdgpu_buffer_rsrc_t po = __builtin_amdgcn_make_buffer_rsrc((void*)(a.part_o + p0 * D), 0, (unsigned)(chunks - 1) * hop + D * 4, 0x00020000);
        auto fetch = [&](int c) {                           // before their weights are known: those of chunks without keys are read and dropped
#pragma unroll
            for (int i = 0; i < FLY; ++i)
                v[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(po, (unsigned)min(c + i * AT + sub, c_hi - 1) * hop + col * 4, 0, 0));
        };
        if (c_lo < c_hi) fetch(c_lo);
        for (int c0 = c_lo; c0 < c_hi; c0 += 64) {
            float m = -INFINITY, ls = 0.f;
            if (c0 + lane < c_hi) { const float2 x = *(const float2*)&a.part_ml[(p0 + (c0 + lane) * step) * 2]; m = x.x; ls = x.y; }
            const float Mn = fmaxf(M, wave_top(m)), ref = Mn == -INFINITY ? 0.f : Mn;
            const float f = __builtin_amdgcn_exp2f(m - ref), old = __builtin_amdgcn_exp2f(M - ref);
            l = l * old + wave_total(ls * f);
            const float w = m == -INFINITY ? -1.f : f;      // (no keys, or no chunk; weights are not negative)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] *= old;
            M = Mn;
            const int cn = min(64, c_hi - c0);
            for (int c = 0; c < cn; c += FLY * AT) {
#pragma unroll
                for (int i = 0; i < FLY; ++i) {
                    float wx = 0.f;
#pragma unroll
                    for (int k = 0; k < AT; ++k) {
                        const float x = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), c + i * AT + k));
                        wx = sub == k ? x : wx;
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[e] += wx == -1.f ? 0.f : v[i][e] * wx;
                }
                if (c0 + c + FLY * AT < c_hi) fetch(c0 + c + FLY * AT);
            }
        }
#pragma unroll
        for (int o = LPR; o < 64; o <<= 1)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor(acc[e], o, 64);
        if constexpr (WAVES == 4) {                          // (one head a workgroup: every wave is here)
            if (lane == 0) { sh_m[wave] = M; sh_l[wave] = l; }
            if (sub == 0) sh_o[wave][lane] = acc;
            __syncthreads();
            if (wave) return;
            M = fmaxf(fmaxf(sh_m[0], sh_m[1]), fmaxf(sh_m[2], sh_m[3]));
            const float ref = M == -INFINITY ? 0.f : M;
            l = 0.f;
            acc = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const float f = __builtin_amdgcn_exp2f(sh_m[x] - ref);
                l += sh_l[x] * f;
                const f32x4 v = sh_o[x][lane % LPR];
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[e] += v[e] * f;
            }
        }
        const float inv = l > 0.f ? (e4m3 && a.v_scale ? a.v_scale[hk] : 1.f) / l : l == 0.f ? 0.f : l;
        if (sub == 0 && col < a.hd)
            *(bf16x4*)(a.out + (long)tok * a.ldo + (long)h * a.hd + col) = (bf16x4){f2bf(acc[0] * inv), f2bf(acc[1] * inv), f2bf(acc[2] * inv), f2bf(acc[3] * inv)};
    }
}

// ---------------------------------------------------------------------------------------------
// Sixteen rows a tile for a token (the G rows of a key-value head), 64 for drafted ones, 128 beyond.  Sixteen requests over 5,000 keys, 28 / 4
// heads of 128, in tiles of 16 / 64 / 128 rows: 2 tokens (14 rows) 38 / 38 / 39 us, 5 (35) 66 / 40 / 41, 9 (63) 66 / 44 / 44, 10 (70) 112 / 47 / 45;
// e4m3, 7 tokens (49): 64 / 128 rows 36.5 / 39.8 us.
static int rows_of_tile(const PagedAttnArgs* a, int max_q) {
    const long rows = (long)(max_q > 0 ? max_q : (a->n_tokens + a->n - 1) / (a->n > 0 ? a->n : 1)) * a->G;
    return rows <= 16 ? 16 : rows <= 64 ? 64 : 128;
}
static int template_dim(const PagedAttnArgs* a) { return a->hd <= 64 ? 64 : 128; }

size_t paged_partial_floats(const PagedAttnArgs* a) { return (size_t)a->target * a->kv_heads * a->tile_rows * template_dim(a); }

static PagedDiv div_by(unsigned d) {
    int s = 0;
    while ((1u << s) < d) ++s;
    return {(unsigned)(((uint64_t)1 << 32) * (((uint64_t)1 << s) - d) / d + 1), s};
}

size_t paged_attention_plan(PagedAttnArgs* a, int n_cus, int max_q, int max_len) {
    const int TR = a->tile_rows = rows_of_tile(a, max_q);
    const long tiles = (long)a->n_tokens * a->G / TR + a->n;              // of one key-value head, at most
    // Two workgroups a CU: what registers and LDS let run at once, and fewer, longer ones leave less to join (four, for tokens, against two:
    // sixteen over 12,000 keys 80.7 / 77.9 us, one over 32,000 29.3 / 22.7 us).
    a->target = (2 * n_cus + a->kv_heads - 1) / a->kv_heads;
    if (a->target > 1000) a->target = 1000;                               // (see TRIES)
    a->inv_target = 1.f / (float)a->target;
    a->by_G = div_by(a->G); a->by_kv_heads = div_by(a->kv_heads); a->by_heads = div_by(a->G * a->kv_heads);
    a->min_blocks = 2;                                                    // 128 keys: a block of 32 for each of four waves (64 keys at least: within 2 % either way)
    long cap = (long)a->max_blocks << a->lps;
    if (max_len > 0 && max_len < cap) cap = max_len;
    const long nb = (cap + 63) / 64;
    // Short sequences are not split, which saves the join and its launch, twice as far where tiles fill half the CUs anyway; us split / whole, heads
    // of 128: one token over 512 keys 13.6 / 11.1, 768 12.8 / 14.0; 64 tokens over 1,024 keys 28.5 / 24.8; 5 over 384 12.9 / 12.2, over 512 12.9 / 14.2;
    // 16 x 36 over 384 27 / 18, one of 40, heads of 64, over 768 13.3 / 18.2; tokens with heads of 64: one over 768 12.7 / 10.4, 128 over 2,048 30 / 23.8.
    const long whole = (TR > 16 ? 6 : a->hd > 64 ? 8 : 16) * (2 * tiles * a->kv_heads >= n_cus ? 2 : 1);
    a->cmax = (int)(nb <= whole ? 1 : nb / a->min_blocks);
    const long by_split = a->target + tiles, by_len = tiles * a->cmax;
    a->grid_items = (int)(by_len < by_split ? by_len : by_split);
    if (a->cmax == 1) return 0;
    return (paged_partial_floats(a) + (size_t)a->target * a->kv_heads * TR * 2) * sizeof(float) + (size_t)a->n * 2 * sizeof(int);
}

template <int D, bool E4M3, int TR>
static hipError_t launch(const PagedAttnArgs* a, hipStream_t st) {
    if constexpr (TR > 16) {
        if (a->precise) paged_tiles_halves(a, E4M3, st);
        else launch_tiles<D, E4M3, TR, false>(a, st);
    } else paged_attn_rows_kernel<D, E4M3><<<a->grid_items * a->kv_heads, 256, 0, st>>>(*a);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && a->cmax > 1) {
        // of many tokens a wave looks at all heads of one: mostly there is nothing to join (8,192 tokens: 5 us, with a wave a head 35 us); of few
        // rows four waves share the chunks (one token over 32,000 keys: 29 us, with one wave 67 us)
        const int heads = a->kv_heads * a->G, each = a->n_tokens >= 2048 ? heads : 1;
        const long rows = (long)a->n_tokens * (heads / each);
        if (rows <= 1024) paged_attn_join_kernel<D, TR, 4><<<(int)rows, 256, 0, st>>>(*a, E4M3, each);
        else paged_attn_join_kernel<D, TR, 1><<<(int)((rows + 3) / 4), 256, 0, st>>>(*a, E4M3, each);
        e = hipGetLastError();
    }
    return e;
}
template <int D, bool E4M3>
static hipError_t launch(const PagedAttnArgs* a, hipStream_t st) {
    return a->tile_rows == 16 ? launch<D, E4M3, 16>(a, st) : a->tile_rows == 64 ? launch<D, E4M3, 64>(a, st) : launch<D, E4M3, 128>(a, st);
}
hipError_t paged_attention(const PagedAttnArgs* a, int e4m3, hipStream_t st) {
    if (template_dim(a) == 64) return e4m3 ? launch<64, true>(a, st) : launch<64, false>(a, st);
    return e4m3 ? launch<128, true>(a, st) : launch<128, false>(a, st);
}
#endif
