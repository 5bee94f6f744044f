// paged.h -- argument records and launchers of the paged key-value cache (paged_tables.hip, paged_append.hip, paged_attention.hip;
// entry points in api_paged.hip).
//
// Keys and values of many sequences live in one pool of pages: [layers][n_pages][kv_heads][page_size][head_dim], so the page_size rows of
// one key-value head are contiguous - the unit one workgroup streams.  page_size is a power of two of at least 16: sixteen consecutive,
// aligned keys (one MFMA tile) are always in one page, and the page lookup is one scalar load per tile.
#pragma once
#include "aha_common.h"

enum { PAGED_BF16 = 0, PAGED_E4M3 = 1 };
// what reserve / truncate put in status[0] (a sum of these); with any of them set nothing was changed
enum { PAGED_NO_PAGES = 1, PAGED_MANY_TOKENS = 2, PAGED_BAD_SEQ = 4, PAGED_TWICE = 8, PAGED_TOO_LONG = 16, PAGED_BAD_COUNT = 32, PAGED_BAD_PAGE = 64 };
#define PAGED_MAX_SEQS 65536                     // sequences of a pool: one bit each in LDS finds a sequence that is listed twice

struct PagedTables {
    int *table, *lens, *free_pages, *n_free;     // [max_seqs][max_blocks], [max_seqs], [n_pages], [1]
    int n_pages, lps, max_seqs, max_blocks;      // lps = log2(page_size)
};

struct PagedReserveArgs {
    PagedTables t;
    const int *seqs, *counts; int n;             // counts: new tokens (reserve) or new lengths (truncate)
    int *slots, *positions; int n_tokens;        // [n_tokens]
    int *cu, *status;                            // [n + 1], [2]
};

struct PagedAppendArgs {
    const bf16 *q, *k, *v; long ldq, ldk, ldv;   // rows of a token; head h at column h * hd
    bf16* q_out; long ldqo;
    void *k_pages, *v_pages;                     // this layer's
    const float *k_scale, *v_scale;              // [kv_heads], E4M3 only
    const int *slots, *positions;
    const bf16 *cos, *sin; int n_pos;            // [n_pos][hd]; null: no rotation
    int n_tokens, heads, kv_heads, hd, lps, n_slots, e4m3;
};

struct PagedDiv { unsigned mul; int shift; };     // n / d = (high word of n * mul, + n) >> shift

struct PagedAttnArgs {
    const bf16* q; long ldq; bf16* out; long ldo;
    const void *k_pages, *v_pages;               // this layer's
    const float *k_scale, *v_scale;
    const int *table, *lens, *seqs, *cu;
    float *part_o, *part_ml;                     // [target][kv_heads][tile rows][D] / [..][2]: partial results
    int* info;                                   // [n][2]: a request's first partial result and its chunks a tile
    int n, n_tokens, max_seqs, max_blocks, n_pages, lps, kv_heads, G, hd, window;
    float scale;
    int target, min_blocks, cmax;                // the split: see schedule() in paged_attention.hip
    float inv_target;
    int most_keys;                               // that a tile's rows see between them
    PagedDiv by_G, by_kv_heads, by_heads;
    int grid_items, tile_rows;                   // workgroups a key-value head; rows of a tile
    int precise;                                 // tiles of many rows: P as two bf16 halves
};

hipError_t paged_reserve(const PagedReserveArgs* a, hipStream_t st);
hipError_t paged_truncate(const PagedReserveArgs* a, hipStream_t st);
hipError_t paged_append(const PagedAppendArgs* a, hipStream_t st);
// fills target / min_blocks / cmax / grid_items for max_len keys at most and returns the bytes of partial results the call needs (0: no split)
size_t paged_attention_plan(PagedAttnArgs* a, int n_cus, int max_q, int max_len);
size_t paged_partial_floats(const PagedAttnArgs* a);          // floats of part_o; part_ml and info lie behind them
hipError_t paged_attention(const PagedAttnArgs* a, int e4m3, hipStream_t st);
void paged_tiles_halves(const PagedAttnArgs* a, int e4m3, hipStream_t st);      // its launch of tiles, with P as two halves
