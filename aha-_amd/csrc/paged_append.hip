// Rotation of new queries and keys, and storage of new keys and values in the pages of their slots.
//
// The pair (x[d], x[d + D/2]) turns by the angle of its token's position (rows of the cos / sin table); the turn is done in fp32 on the bf16
// inputs and rounded once, to bf16 or, for an 8-bit cache, x / scale clamped to +-448 to e4m3 (products of two bf16 values are exact in fp32,
// so the sum is the only other rounding).  A thread owns eight pairs: 16-byte loads and stores, the table row comes from the L1.  Bound by the bytes:
// 19,000 tokens of 28 / 4 heads of 128 (356 MB) 69 us, 5.1 TB/s (a large copy: 4.9), into e4m3 pages (336 MB) 67; 16 tokens 3.4 us, a launch.
#include "paged.h"

static __device__ __forceinline__ unsigned pack4_e4m3(float a, float b, float c, float d) {
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, p, true);
}
// NaN stays NaN (both comparisons are false)
static __device__ __forceinline__ float clamp448(float x) { return x > 448.f ? 448.f : x < -448.f ? -448.f : x; }

template <bool E4M3>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendArgs a) {
    const int half = a.hd >> 1, C = half >> 3;                 // chunks of eight pairs a head
    const int rows = a.heads + 2 * a.kv_heads, per = rows * C;
    const long id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= (long)per * a.n_tokens) return;
    const int tok = (int)(id / per), rem = (int)(id - (long)tok * per);
    const int row = rem / C, c = (rem - row * C) * 8;
    const bool is_q = row < a.heads, is_k = !is_q && row < a.heads + a.kv_heads;
    const int h = is_q ? row : is_k ? row - a.heads : row - a.heads - a.kv_heads;
    const bf16* src = (is_q ? a.q + tok * a.ldq : is_k ? a.k + tok * a.ldk : a.v + tok * a.ldv) + h * a.hd + c;
    const bf16x8 x1 = *(const bf16x8*)src, x2 = *(const bf16x8*)(src + half);
    float y1[8], y2[8];
    if (a.cos && (is_q || is_k)) {
        const int pos = min(max(a.positions[tok], 0), a.n_pos - 1);
        const long t = (long)pos * a.hd + c;
        const bf16x8 c1 = *(const bf16x8*)(a.cos + t), c2 = *(const bf16x8*)(a.cos + t + half);
        const bf16x8 s1 = *(const bf16x8*)(a.sin + t), s2 = *(const bf16x8*)(a.sin + t + half);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            y1[e] = bf2f(x1[e]) * bf2f(c1[e]) - bf2f(x2[e]) * bf2f(s1[e]);
            y2[e] = bf2f(x2[e]) * bf2f(c2[e]) + bf2f(x1[e]) * bf2f(s2[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) { y1[e] = bf2f(x1[e]); y2[e] = bf2f(x2[e]); }
    }
    if (is_q || !E4M3) {
        bf16* dst;
        if (is_q) dst = a.q_out + tok * a.ldqo + h * a.hd + c;
        else {
            const int slot = a.slots[tok];
            if ((unsigned)slot >= (unsigned)a.n_slots) return;
            const long page = slot >> a.lps;
            dst = (bf16*)(is_k ? a.k_pages : a.v_pages) + (((page * a.kv_heads + h) << a.lps) + (slot & ((1 << a.lps) - 1))) * a.hd + c;
        }
        bf16x8 o1, o2;
#pragma unroll
        for (int e = 0; e < 8; ++e) { o1[e] = f2bf(y1[e]); o2[e] = f2bf(y2[e]); }
        *(bf16x8*)dst = o1;
        *(bf16x8*)(dst + half) = o2;
    } else {
        const int slot = a.slots[tok];
        if ((unsigned)slot >= (unsigned)a.n_slots) return;
        const float* sc = is_k ? a.k_scale : a.v_scale;
        const float s = sc ? sc[h] : 1.f;
        const long page = slot >> a.lps;
        uint8_t* dst = (uint8_t*)(is_k ? a.k_pages : a.v_pages) + (((page * a.kv_heads + h) << a.lps) + (slot & ((1 << a.lps) - 1))) * a.hd + c;
        const float by = s == 0.f ? 1.f : s, keep = s == 0.f ? 0.f : 1.f;      // a scale of 0 stores 0 (x / 0 would be 448 or no number); NaN stays NaN
#pragma unroll
        for (int e = 0; e < 8; ++e) { y1[e] = clamp448(y1[e] / by) * keep; y2[e] = clamp448(y2[e] / by) * keep; }
        *(uint2*)dst = make_uint2(pack4_e4m3(y1[0], y1[1], y1[2], y1[3]), pack4_e4m3(y1[4], y1[5], y1[6], y1[7]));
        *(uint2*)(dst + half) = make_uint2(pack4_e4m3(y2[0], y2[1], y2[2], y2[3]), pack4_e4m3(y2[4], y2[5], y2[6], y2[7]));
    }
}

hipError_t paged_append(const PagedAppendArgs* a, hipStream_t st) {
    const long work = (long)a->n_tokens * (a->heads + 2 * a->kv_heads) * (a->hd / 16);
    const unsigned grid = (unsigned)((work + 255) / 256);
    if (a->e4m3) paged_append_kernel<true><<<grid, 256, 0, st>>>(*a);
    else paged_append_kernel<false><<<grid, 256, 0, st>>>(*a);
    return hipGetLastError();
}
