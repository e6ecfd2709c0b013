// Attention over a cache of 8 bits for portions of prompts: tiles of rows on the matrix cores.
#include "scaled_attend.h"

#include <algorithm>

namespace {

constexpr int MOST_ROWS = 65535 * 16;                   // of a portion in one launch
constexpr int MOST_REACH = 2147483647 - 2 * MOST_ROWS;   // positions, the rows of a block that a portion does not have among them, are numbers of 32 bits

// Portions of prompts: a block per (request, head, tile of rows). SPLITS of its four waves take the tiles of keys in turn, each with statistics of
// its own, and meet in LDS; with two, the other two do the same for 16 CT rows more, at the same time, so that half of what they read comes from
// the compute unit's own cache. Tiles with the most keys of all heads come first.
template <typename T, int HD, int CT, int SPLITS, bool WHOLE>
__global__ __launch_bounds__(256, HD == 256 ? 1 : 2) void scaled_tiles_attention_kernel(AttendArguments a) {
    constexpr bool WIDE = sizeof(T) == 4;
    typedef ScaledSweep<HD, CT, WIDE, true, WHOLE> Sweep;
    constexpr int WAVES = 4, GROUPS = WAVES / SPLITS, WAVE_ROWS = 16 * CT, ROWS = GROUPS * WAVE_ROWS;
    // the queries' operands while keys are walked; then what the waves hold, row by row
    constexpr int PITCH = HD + 4;
    __shared__ union {
        bf16x8 queries[GROUPS][Sweep::Q_PIECES];
        float meeting[WAVES][WAVE_ROWS][PITCH];
    } lds;
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), group = wave % GROUPS, split = wave / GROUPS;
    const int request = blockIdx.z, head = blockIdx.x, head_size = a.planes.head_size;
    const int q_first = a.q_starts[request], q_len = min(a.q_starts[request + 1], a.n_rows) - q_first;
    const int row0 = (gridDim.y - 1 - blockIdx.y) * ROWS;
    const int reach = (int)min((long long)a.max_blocks << a.planes.page_shift, (long long)MOST_REACH) - 1;
    const int context = min(a.context_lens[request], reach);
    if (row0 >= q_len || context < 0 || q_first < 0) return;   // (a negative context: a padding request, whose rows are nobody's)
    const int kv_head = head / (a.n_heads / a.planes.n_kv_heads);
    const int own0 = row0 + group * WAVE_ROWS;   // the wave's first row, if the portion has it
    const int position0 = min(context + own0, reach), position1 = min(context + min(own0 + WAVE_ROWS, q_len) - 1, reach);

    Sweep sweep;
    sweep.init(head_size, lane);
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        const int local = own0 + 16 * ct + lane % 16;
        const bool valid = local < q_len;
        if (ct % SPLITS == split) {
            sweep.template load_query<T>(ct, valid ? static_cast<const T*>(a.q) + (size_t)(q_first + local) * a.q_stride + head * head_size : nullptr, head_size, a.aligned, a.negative, lane);
            sweep.share_query(ct, lds.queries[group], lane);
        }
    }
    sweep.q_shared = lds.queries[group];
    __syncthreads();
    if (GROUPS == 1 || own0 < q_len) {
        const TileRange range(scaled_first_key(position0, a.window, a.chunk), position1, a.keep);
        sweep.tiles(range, split, SPLITS, range.count, a.block_tables + (size_t)request * a.max_blocks, a.planes, kv_head, a.scale,
                    {context + own0 + lane % 16, position1, a.window, a.chunk, a.keep}, scaled_first_key(position1, a.window, a.chunk), position0, lane);
    }

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
        const int of_group = GROUPS == 1 ? 0 : row / WAVE_ROWS, at = GROUPS == 1 ? row : row % WAVE_ROWS;
        float top = NO_SCORE;
#pragma unroll
        for (int w = 0; w < SPLITS; w++) top = fmaxf(top, lds.meeting[w * GROUPS + of_group][at][HD]);
        float total = a.sinks ? weight_of<WIDE>(a.sinks[head] * a.sink_factor - top) : 0.0f;
        f32x4 value = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < SPLITS; w++) {
            const float* const part = lds.meeting[w * GROUPS + of_group][at];
            const float factor = weight_of<WIDE>(part[HD] - top);
            total += part[HD + 1] * factor;
            const f32x4 theirs = *reinterpret_cast<const f32x4*>(part + d);
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
