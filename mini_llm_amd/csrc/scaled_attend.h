// What the two kernels of attention over a cache of 8 bits share (scaled_attention_rows.hip, scaled_attention_tiles.hip): their arguments and what refuses them,
// and how results are written.
//
// A token at position p attends to the keys max(0, p - window + 1) .. p of its request (window 0: all; with kept first keys also to those;
// or, with chunks, to the keys of its own chunk up to p). A row without a request, or at a position before the first, sees nothing:
// zeros.
#pragma once

#include "scaled_sweep.h"

struct AttendArguments {
    const void* q;
    long long q_stride;
    void* out;
    long long out_stride;
    const int* token_request;
    const int* positions;
    const int* q_starts;
    const int* context_lens;
    const int* block_tables;
    const float* sinks;
    ScaledPlanes planes;
    int max_blocks, n_tables, n_rows, n_heads, window, chunk, keep, aligned, negative, wide_out, out_packed, out_aligned;
    ScoreScale scale;
    float sink_factor;   // log2 e where weights are powers of two
};

// One result: of row `row`, element `at` of its n_heads * head_size.
template <typename T>
__device__ __forceinline__ void put_result(const AttendArguments& a, int row, int at, float value) {
    const size_t index = a.out_packed ? packed_element<T>(row, at, a.n_heads * a.planes.head_size) : (size_t)row * a.out_stride + at;
    if (sizeof(T) == 4 || !a.wide_out) static_cast<T*>(a.out)[index] = from_float<T>(value);
    else static_cast<float*>(a.out)[index] = value;
}

// Four neighbouring results of a row that is not packed.
template <typename T>
__device__ __forceinline__ void put_four(const AttendArguments& a, int row, int at, f32x4 value) {
    const size_t index = (size_t)row * a.out_stride + at;
    if (sizeof(T) == 4 || a.wide_out) {
        float* const to = static_cast<float*>(a.out) + index;
        if (a.out_aligned) *reinterpret_cast<f32x4*>(to) = value;
        else
            for (int e = 0; e < 4; e++) to[e] = value[e];
    } else {
        bf16_t* const to = static_cast<bf16_t*>(a.out) + index;
        const bf16x4 rounded = {static_cast<bf16_t>(value[0]), static_cast<bf16_t>(value[1]), static_cast<bf16_t>(value[2]), static_cast<bf16_t>(value[3])};
        if (a.out_aligned) *reinterpret_cast<bf16x4*>(to) = rounded;
        else
            for (int e = 0; e < 4; e++) to[e] = rounded[e];
    }
}

// What a row sees, or no tile at all.
struct RowView {
    int request, position, first;
    __device__ __forceinline__ RowView(const AttendArguments& a, int row) {
        request = a.token_request[row];
        position = a.positions[row];
        if (request >= a.n_tables) request = -1;
        position = min(position, (int)min((long long)a.max_blocks << a.planes.page_shift, 2147483647LL) - 1);
        first = scaled_first_key(max(position, 0), a.window, a.chunk);
    }
    __device__ __forceinline__ bool sees() const { return request >= 0 && position >= 0; }
};

inline int refuse_attend(const char* what, const AttendArguments& a, int page_size, int dtype) {
    const ScaledPlanes& p = a.planes;
    MLLM_REQUIRE(a.n_rows >= 0 && a.n_heads > 0 && p.n_kv_heads > 0 && a.max_blocks > 0 && a.n_tables > 0 && p.num_pages > 0, "%s: bad sizes", what);
    MLLM_REQUIRE(a.n_heads % p.n_kv_heads == 0, "%s: %d heads do not divide into %d key/value heads", what, a.n_heads, p.n_kv_heads);
    MLLM_REQUIRE(p.head_size > 0 && p.head_size % 16 == 0 && p.head_size <= SCALED_MAX_HEAD, "%s: heads of %d (a multiple of 16 up to %d)", what, p.head_size, SCALED_MAX_HEAD);
    MLLM_REQUIRE(page_size >= BLOCK_TOKENS && (page_size & (page_size - 1)) == 0, "%s: page size %d is no power of two of at least %d", what, page_size, BLOCK_TOKENS);
    MLLM_REQUIRE(dtype == MLLM_F32 || dtype == MLLM_BF16, "%s: unknown dtype %d", what, dtype);
    MLLM_REQUIRE(a.window >= 0 && a.chunk >= 0 && !(a.window && a.chunk), "%s: bad window or chunk", what);
    MLLM_REQUIRE(a.keep >= 0 && (a.keep == 0 || a.window > 0), "%s: first keys are kept beside a window", what);
    MLLM_REQUIRE(a.q_stride >= (long long)a.n_heads * p.head_size && a.out_stride >= (long long)a.n_heads * p.head_size, "%s: rows are too short for the heads", what);
    MLLM_REQUIRE(!(a.wide_out && a.out_packed), "%s: rows in the packed layout leave in the queries' type", what);
    return 0;
}

inline AttendArguments attend_arguments(const void* q, long long q_stride, const void* k_codes, const float* k_scales, const void* v_codes, const float* v_scales, void* out,
                                 long long out_stride, const int* block_tables, int max_blocks, int n_tables, int num_pages, int n_rows, int n_heads, int n_kv_heads,
                                 int head_size, int page_size, int window, float scale, int dtype, float softcap, const float* sinks, int chunk, int keep, int wide_out) {
    int shift = 0;
    while ((1 << shift) < page_size) shift++;
    const float unit = dtype == MLLM_F32 ? 1.0f : 1.4426950408889634f, size = scale < 0.0f ? -scale : scale;
    AttendArguments a = {};
    a.q = q, a.q_stride = q_stride, a.out = out, a.out_stride = out_stride, a.block_tables = block_tables, a.sinks = sinks;
    a.planes = {(const uint8_t*)k_codes, k_scales, (const uint8_t*)v_codes, v_scales, num_pages, n_kv_heads, head_size, shift};
    a.max_blocks = max_blocks, a.n_tables = n_tables, a.n_rows = n_rows, a.n_heads = n_heads, a.window = window, a.chunk = chunk, a.keep = keep;
    a.aligned = (uintptr_t)q % 16 == 0 && q_stride * (dtype == MLLM_F32 ? 4 : 2) % 16 == 0;
    const int out_size = dtype == MLLM_F32 || wide_out ? 4 : 2;
    a.out_aligned = (uintptr_t)out % (4 * out_size) == 0 && out_stride % 4 == 0;   // four results at a time
    a.negative = scale < 0.0f, a.wide_out = wide_out;
    // (a factor of zero would make numbers that are none of masked scores: 1e-30 leaves as little between any two others)
    a.scale = {size * unit > 1e-30f ? size * unit : 1e-30f, softcap > 0.0f ? size / softcap : 0.0f, softcap > 0.0f ? softcap * unit : 0.0f};
    a.sink_factor = unit;
    return a;
}
