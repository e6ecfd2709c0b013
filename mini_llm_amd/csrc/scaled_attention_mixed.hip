// Attention over a cache of 8 bits for a step of both kinds, decoding rows beside portions of prompts, in one launch.
#include "scaled_attend.h"

namespace {

// The blocks of rows first, then those of tiles of rows, each as in its own kernel: either part's wait for its longest block runs under the other's blocks
// (33 rows beside three portions, float32, 12 heads of 64: 24.5 us in two launches, 16.4 in one).
template <typename T, int HD, int CT, bool WHOLE>
__global__ __launch_bounds__(256, 2) void scaled_mixed_attention_kernel(AttendArguments a, int short_rows, int sets, int n_runs, int run_tiles, float* __restrict__ parts,
                                                                        int short_requests, int n_tiles) {
    __shared__ union {
        TileMemory<T, HD, CT, 4> tile;
        float meeting[4 * 16 * (HD + 4)];
    } lds;
    const int row_blocks = short_rows * sets * n_runs;
    int block = blockIdx.x;
    if (block < row_blocks) {
        const int row = block % short_rows;
        block /= short_rows;
        attend_row<T, HD, WHOLE>(a, row, block % sets, block / sets, 4, run_tiles, n_runs, parts, lds.meeting);
    } else {
        block -= row_blocks;
        const int head = block % a.n_heads;
        block /= a.n_heads;
        attend_tile<T, HD, CT, 4, WHOLE>(a, short_requests + block / n_tiles, head, n_tiles - 1 - block % n_tiles, lds.tile);
    }
}

}  // namespace

// The first short_rows rows, of the first short_requests requests, by themselves (mllm_scaled_attention_rows, by four waves), the rows of the other requests
// as portions (mllm_scaled_attention_tiles). q_starts, context_lens and block_tables are of all requests.
MLLM_API int mllm_scaled_attention_mixed(const void* q, long long q_stride, const void* k_codes, const float* k_scales, const void* v_codes, const float* v_scales, void* out,
                                         long long out_stride, const int* token_request, const int* positions, const int* q_starts, const int* context_lens,
                                         const int* block_tables, int max_blocks, int n_tables, int num_pages, int n_rows, int n_heads, int n_kv_heads, int head_size,
                                         int page_size, int window, float scale, int dtype, float softcap, const float* sinks, int chunk, int keep, int wide_out, int short_rows,
                                         int short_requests, int n_requests, int max_q_len, int run_tiles, int n_runs, float* parts, hipStream_t stream) {
    AttendArguments a = attend_arguments(q, q_stride, k_codes, k_scales, v_codes, v_scales, out, out_stride, block_tables, max_blocks, n_tables, num_pages, n_rows, n_heads,
                                         n_kv_heads, head_size, page_size, window, scale, dtype, softcap, sinks, chunk, keep, wide_out);
    a.token_request = token_request, a.positions = positions, a.q_starts = q_starts, a.context_lens = context_lens;
    if (int status = refuse_attend("scaled_attention_mixed", a, page_size, dtype)) return status;
    MLLM_REQUIRE(head_size <= 128, "scaled_attention_mixed: heads of %d (up to 128)", head_size);
    MLLM_REQUIRE(short_rows > 0 && short_rows < n_rows && short_requests > 0 && short_requests < n_requests && n_requests <= n_tables && max_q_len > 0 && max_q_len <= MOST_ROWS,
                 "scaled_attention_mixed: %d of %d rows and %d of %d requests do not cut the batch in two", short_rows, n_rows, short_requests, n_requests);
    MLLM_REQUIRE(run_tiles >= 1 && n_runs >= 1 && n_runs <= MOST_RUNS && (n_runs == 1 || parts != nullptr), "scaled_attention_mixed: runs of %d tiles, %d runs (with memory for more than one)",
                 run_tiles, n_runs);
    const int sets = n_kv_heads * ceil_div(n_heads / n_kv_heads, 16), tile_rows = head_size <= 64 && dtype == MLLM_BF16 ? 32 : 16, n_tiles = ceil_div(max_q_len, tile_rows);
    const long long blocks = (long long)short_rows * sets * n_runs + (long long)n_heads * n_tiles * (n_requests - short_requests);
    MLLM_REQUIRE(blocks < 2147483648LL / 256, "scaled_attention_mixed: too many blocks for one launch");
    mllm_count_kernel(MLLM_K_SCALED_ATTENTION_MIXED);
#define MIXED_CASE(T, HD, CT)                                                                                                                                              \
    {                                                                                                                                                                      \
        if (page_size >= TILE_KEYS) scaled_mixed_attention_kernel<T, HD, CT, true><<<(int)blocks, 256, 0, stream>>>(a, short_rows, sets, n_runs, run_tiles, parts, short_requests, n_tiles); \
        else scaled_mixed_attention_kernel<T, HD, CT, false><<<(int)blocks, 256, 0, stream>>>(a, short_rows, sets, n_runs, run_tiles, parts, short_requests, n_tiles);              \
    }
    if (dtype == MLLM_F32) {
        if (head_size <= 64) MIXED_CASE(float, 64, 1)
        else MIXED_CASE(float, 128, 1)
    } else {
        if (head_size <= 64) MIXED_CASE(bf16_t, 64, 2)
        else MIXED_CASE(bf16_t, 128, 1)
    }
#undef MIXED_CASE
    if (int status = mllm_check_launch("scaled_attention_mixed")) return status;
    return n_runs == 1 ? 0 : scaled_merge(a, dtype, short_rows, run_tiles, n_runs, parts, stream);
}
