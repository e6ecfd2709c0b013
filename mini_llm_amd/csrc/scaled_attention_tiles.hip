// Attention over a cache of 8 bits for portions of prompts: tiles of rows on the matrix cores.
#include "scaled_attend.h"

#include <algorithm>

namespace {

constexpr int MOST_ROWS = 65535 * 16;                   // of a portion in one launch
constexpr int MOST_REACH = 2147483647 - 2 * MOST_ROWS;   // positions, the rows of a block that a portion does not have among them, are numbers of 32 bits

// Portions of prompts: a block per (request, head, tile of 16 CT rows), whose waves hold all those rows and take the tiles of keys in turn,
// each with statistics of its own, and meet in LDS. Tiles with the most keys come first.
template <typename T, int HD, int CT, bool WHOLE>
__global__ __launch_bounds__(256, HD == 256 ? 1 : 2) void scaled_tiles_attention_kernel(AttendArguments a) {
    constexpr bool WIDE = sizeof(T) == 4;
    typedef ScaledSweep<HD, CT, WIDE, true, WHOLE> Sweep;
    constexpr int ROWS = 16 * CT, WAVES = 4;
    // the queries' operands while keys are walked; then what the waves hold, row by row
    constexpr int PITCH = HD + 4;
    __shared__ union {
        bf16x8 queries[Sweep::Q_PIECES];
        float meeting[WAVES][ROWS][PITCH];
    } lds;
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int request = blockIdx.z, head = blockIdx.x, head_size = a.planes.head_size;
    const int q_first = a.q_starts[request], q_len = min(a.q_starts[request + 1], a.n_rows) - q_first;
    const int row0 = (gridDim.y - 1 - blockIdx.y) * ROWS;
    const int reach = (int)min((long long)a.max_blocks << a.planes.page_shift, (long long)MOST_REACH) - 1;
    const int context = min(a.context_lens[request], reach);
    if (row0 >= q_len || context < 0 || q_first < 0) return;   // (a negative context: a padding request, whose rows are nobody's)
    const int kv_head = head / (a.n_heads / a.planes.n_kv_heads);
    const int position0 = min(context + row0, reach), position1 = min(context + min(row0 + ROWS, q_len) - 1, reach);

    Sweep sweep;
    sweep.init(head_size, lane);
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        const int local = row0 + 16 * ct + lane % 16;
        const bool valid = local < q_len;
        if (ct % WAVES == wave) {
            sweep.template load_query<T>(ct, valid ? static_cast<const T*>(a.q) + (size_t)(q_first + local) * a.q_stride + head * head_size : nullptr, head_size, a.aligned, a.negative, lane);
            sweep.share_query(ct, lds.queries, lane);
        }
    }
    sweep.q_shared = lds.queries;
    __syncthreads();
    const TileRange range(scaled_first_key(position0, a.window, a.chunk), position1, a.keep);
    sweep.tiles(range, wave, WAVES, range.count, a.block_tables + (size_t)request * a.max_blocks, a.planes, kv_head, a.scale,
                {context + row0 + lane % 16, position1, a.window, a.chunk, a.keep}, scaled_first_key(position1, a.window, a.chunk), position0, lane);

    __syncthreads();   // (all waves are through with the queries)
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        float* const mine = lds.meeting[wave][16 * ct + lane % 16];
#pragma unroll
        for (int dt = 0; dt < Sweep::DT; dt++) *reinterpret_cast<f32x4*>(mine + 16 * dt + 4 * (lane / 16)) = sweep.o[ct][dt];
        const float sum = sweep.weight_sum(ct);
        if (lane < 16) {
            mine[HD] = sweep.m[ct];
            mine[HD + 1] = sum;
        }
    }
    __syncthreads();
    // four elements of a row a thread, as they lie in the results
    const int fours = head_size / 4;
    for (int i = threadIdx.x; i < ROWS * fours; i += blockDim.x) {
        const int row = i / fours, d = 4 * (i % fours);
        if (row0 + row >= q_len) break;
        float top = NO_SCORE;
#pragma unroll
        for (int w = 0; w < WAVES; w++) top = fmaxf(top, lds.meeting[w][row][HD]);
        float total = a.sinks ? weight_of<WIDE>(a.sinks[head] * a.sink_factor - top) : 0.0f;
        f32x4 value = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            const float factor = weight_of<WIDE>(lds.meeting[w][row][HD] - top);
            total += lds.meeting[w][row][HD + 1] * factor;
            const f32x4 theirs = *reinterpret_cast<const f32x4*>(&lds.meeting[w][row][d]);
#pragma unroll
            for (int e = 0; e < 4; e++) value[e] += theirs[e] * factor;
        }
        const float inverse = 1.0f / total;
        put_four<T>(a, q_first + row0 + row, head * head_size + d, value * inverse);
    }
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
    const bool half = n_heads * std::min(by_rows, by_longest) < 320;
#define TILES_CASE(T, HD, CT)                                                                                   \
    {                                                                                                           \
        const dim3 grid(n_heads, ceil_div(max_q_len, 16 * CT), n_requests);                                     \
        if (page_size >= TILE_KEYS) scaled_tiles_attention_kernel<T, HD, CT, true><<<grid, 256, 0, stream>>>(a); \
        else scaled_tiles_attention_kernel<T, HD, CT, false><<<grid, 256, 0, stream>>>(a);                       \
    }
    if (dtype == MLLM_F32) {
        if (head_size > 128) TILES_CASE(float, 256, 1)
        else if (head_size > 64) TILES_CASE(float, 128, 1)
        else if (half) TILES_CASE(float, 64, 1)
        else TILES_CASE(float, 64, 2)
    } else if (head_size > 128) TILES_CASE(bf16_t, 256, 1)
    else if (head_size > 64) {
        if (half) TILES_CASE(bf16_t, 128, 1)
        else TILES_CASE(bf16_t, 128, 2)
    } else if (half) TILES_CASE(bf16_t, 64, 2)
    else TILES_CASE(bf16_t, 64, 4)
#undef TILES_CASE
    return mllm_check_launch("scaled_attention_tiles");
}
