// Device-side parameters and launchers of the 8-bit serving kernels (kv8.hip, kv8_attend.hip, f8.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace tsfm {

constexpr int kKvBlock = 64;                // tokens of a cache block (TSFM_KV8_BLOCK)
constexpr int kCodeE4m3 = 0, kCodeI8 = 1;   // TSFM_CODE_*

// tsfm_kv8_cache on the device.
struct Kv8 {
    uint8_t* k;        // (blocks, heads, 64, D)
    uint8_t* v;        // (blocks, heads, D, 64), token 32c + 16a + 4g + i at byte 16g + 8c + 4a + i
    float* scales;     // (blocks, heads, 2)
    uint16_t* k_tail;  // (requests, heads, 64, D)
    uint16_t* v_tail;
    const int32_t* table;  // (requests, width)
    const int32_t* len;    // (requests)
    int32_t requests, heads, blocks, width;
};

struct Kv8Plan {
    const int32_t *n_new, *len, *free_list, *free_count;
    int32_t *len_out, *free_count_out, *table, *cu_tokens, *cu_blocks, *cu_items, *pos, *items, *status;
    int64_t* slots;
    int32_t requests, blocks, width, max_tokens, max_items;
};
hipError_t launch_kv8_plan(const Kv8Plan& p, hipStream_t s);

struct Kv8Release {
    const uint8_t* drop;
    int32_t *len, *table, *free_list, *free_count, *status;
    int32_t requests, blocks, width;
};
hipError_t launch_kv8_release(const Kv8Release& p, hipStream_t s);

struct Kv8Append {
    Kv8 c;
    const int32_t *cu_tokens, *items;
    const uint16_t *k, *v;
    int64_t k_tok, v_tok;
    int32_t max_tokens, max_items;
};
hipError_t launch_kv8_append(const Kv8Append& p, int code, bool bf16, int head_dim, hipStream_t s);

struct Kv8Attend {
    Kv8 c;
    const int32_t* cu_tokens;
    const uint16_t* q;
    uint16_t* o;
    int64_t q_tok, o_tok;
    int32_t heads, max_tokens;
    int32_t group;     // heads / kv heads
    float c2;          // scale * log2(e)
    // Set by kv8_attend_plan: the split of the keys.
    int32_t tiles;     // row tiles per (request, kv head) in the grid
    int32_t chunk;     // cache blocks per workgroup
    int32_t chunks;    // workgroups along the keys, per row tile
    int32_t rows;      // rows of a tile
    int32_t kernel;    // kAttend*
    int32_t once;      // the keys are read past the caches
    int32_t longest_first;  // workgroups take the requests (64 at most) by length
    float* part;       // partial results: O (rows of o, heads, chunks, D), then (max, sum) pairs
};
constexpr int kAttendFew = 0, kAttendMany = 1;
// Picks kernel and split from the sizes and hints; returns the bytes of partial results.
int64_t kv8_attend_plan(Kv8Attend& p, int head_dim, int max_new, int max_len, int cus);
hipError_t launch_kv8_attend(const Kv8Attend& p, int code, bool bf16, int head_dim, hipStream_t s);

struct F8Quantize {
    const void* x;
    uint8_t* codes;
    float* scales;
    int64_t x_ld, codes_ld, scales_ld;
    int32_t rows, cols, group_rows;
};
hipError_t launch_f8_quantize(const F8Quantize& p, int dtype, hipStream_t s);

struct F8Gemm {
    const uint8_t *a, *b;
    const float *a_scales, *b_scales;
    void* c;
    int64_t a_ld, b_ld, a_scales_ld, b_scales_ld, c_ld;
    int32_t m, n, k;
};
hipError_t launch_f8_gemm(const F8Gemm& p, int out_dtype, int cus, hipStream_t s);

}  // namespace tsfm
