// Attention over a cache of 8 bits for portions of prompts: tiles of rows on the matrix cores.
#include "scaled_attend.h"

#include <algorithm>

namespace {

// A block per (request, head, tile of rows). Tiles with the most keys of all heads come first. What bounds it: a wave issues its own conversions, softmax
// arithmetic and products one behind the other, and two waves a SIMD (what 250 registers leave) overlap in part: 16 heads of 128 on 8,192 rows (64 a block, two waves on each half) 281 us, 980 TFLOP/s
// of the keys that are seen (vector instructions in half the cycles, matrix instructions in 46 %); without the exponentials it would be 2 to 5 % less, without the reads of keys and values 23 %.
// 12 heads of 64 on 2,048 rows 21 us, where the launch is one round of blocks and the longest has eight tiles of keys a wave (without the exponentials 19.7, without the reads 20.1); this form, 64 rows
// of heads of up to 64, takes all 256 registers and spills 5 (27 over pages of 16 or 32 tokens).
template <typename T, int HD, int CT, int SPLITS, bool WHOLE>
__global__ __launch_bounds__(256, HD == 256 ? 1 : 2) void scaled_tiles_attention_kernel(AttendArguments a) {
    __shared__ TileMemory<T, HD, CT, SPLITS> lds;
    attend_tile<T, HD, CT, SPLITS, WHOLE>(a, blockIdx.z, blockIdx.x, gridDim.y - 1 - blockIdx.y, lds);
}

}  // namespace

// Portions: the rows of request r are q_starts[r] .. q_starts[r + 1] - 1, the first of them at position context_lens[r] (negative: nobody's rows).
MLLM_API int mllm_scaled_attention_tiles(const void* q, long long q_stride, const void* k_codes, const float* k_scales, const void* v_codes, const float* v_scales, void* out,
                                         long long out_stride, const int* q_starts, const int* context_lens, const int* block_tables, int max_blocks, int n_requests,
                                         int num_pages, int n_rows, int max_q_len, int n_heads, int n_kv_heads, int head_size, int page_size, int window, float scale, int dtype,
                                         float softcap, const float* sinks, int chunk, int keep, int wide_out, hipStream_t stream) {
    AttendArguments a = attend_arguments(q, q_stride, k_codes, k_scales, v_codes, v_scales, out, out_stride, block_tables, max_blocks, n_requests, num_pages, n_rows, n_heads,
                                         n_kv_heads, head_size, page_size, window, scale, dtype, softcap, sinks, chunk, keep, wide_out);
    a.q_starts = q_starts, a.context_lens = context_lens;
    if (int status = refuse_attend("scaled_attention_tiles", a, page_size, dtype)) return status;
    MLLM_REQUIRE(n_requests <= 65535 && max_q_len <= MOST_ROWS, "scaled_attention_tiles: too many requests or rows for one launch");
    if (n_rows == 0 || max_q_len <= 0) return 0;
    mllm_count_kernel(MLLM_K_SCALED_ATTENTION_TILES);
    // Rows a block: as many as the registers hold the sums of (a key is converted once for all of them), or half as many where that leaves fewer
    // blocks than the chip takes at once. us with the whole / half the rows, bfloat16: 12 heads of 64, 512 rows (96 / 192 blocks) 10.1 / 7.4, behind 1,536
    // keys 19.5 / 13.3, 1,024 (192) 13.6 / 10.2, 2,048 (384) 21.7 / 21.6, 8,192 143 / 164; four requests of 512 (384) 14.4 / 15.5; 25 heads, 2,048 (800) 35.1 / 38.4;
    // 16 heads of 128, 512 rows (256) 9.7 / 8.3, 2,048 (1,024) 35.4 / 47.0; in 32-bit 12 heads of 64, 512 rows 10.5 / 8.7, 2,048 (768) 38.7 / 38.3.
    const int whole = dtype == MLLM_F32 ? (head_size <= 64 ? 2 : 1) : head_size <= 64 ? 4 : head_size <= 128 ? 2 : 1;
    const long long by_rows = n_rows / (16 * whole) + n_requests, by_longest = (long long)n_requests * ceil_div(max_q_len, 16 * whole);
    const long long blocks = n_heads * std::min(by_rows, by_longest);
    const bool half = blocks < 320;
    // Heads of 65 to 128, twice the rows a block (half the waves on each) where there are blocks in plenty: us with 32 / 64 rows, 16 heads of 128 on 2,048 rows (1,024 / 512
    // blocks) 35.8 / 36.4, 32 on 1,024 behind 3,072 keys (1,024 / 512) 83.9 / 82.8, 16 on 8,192 (4,096 / 2,048) 299 / 285. (Of 64, on 8,192: 144 / 151.)
    const bool twice = blocks >= 2048;
#define TILES_CASE(T, HD, CT, S)                                                                                   \
    {                                                                                                              \
        const dim3 grid(n_heads, ceil_div(max_q_len, 16 * CT * (4 / S)), n_requests);                              \
        if (page_size >= TILE_KEYS) scaled_tiles_attention_kernel<T, HD, CT, S, true><<<grid, 256, 0, stream>>>(a); \
        else scaled_tiles_attention_kernel<T, HD, CT, S, false><<<grid, 256, 0, stream>>>(a);                       \
    }
    if (dtype == MLLM_F32) {
        if (head_size > 128) TILES_CASE(float, 256, 1, 4)
        else if (head_size > 64) TILES_CASE(float, 128, 1, 4)
        else if (half) TILES_CASE(float, 64, 1, 4)
        else TILES_CASE(float, 64, 2, 4)
    } else if (head_size > 128) TILES_CASE(bf16_t, 256, 1, 4)
    else if (head_size > 64) {
        if (half) TILES_CASE(bf16_t, 128, 1, 4)
        else if (twice) TILES_CASE(bf16_t, 128, 2, 2)
        else TILES_CASE(bf16_t, 128, 2, 4)
    } else if (half) TILES_CASE(bf16_t, 64, 2, 4)
    else TILES_CASE(bf16_t, 64, 4, 4)
#undef TILES_CASE
    return mllm_check_launch("scaled_attention_tiles");
}
