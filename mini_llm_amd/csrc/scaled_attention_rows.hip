// Attention over a cache of 8 bits for rows by themselves: decoding, short portions, and whatever else comes without the shape of portions.
#include "scaled_attend.h"

namespace {

// The most waves a block of rows may have: as many as have the registers they need.
constexpr int rows_waves(int padded, int size) { return padded == 64 ? (size == 2 ? 16 : 8) : 1024 / padded; }

// A block per row, set of heads and run of keys. What bounds it is the cache's bytes, 2 (head_size + 0.25) a key for all
// heads of a set together: 16 rows at 20,000 to 32,000 keys of 8 heads of 128 (32 query heads) 142 us for 810 MB, 5.7 TB/s; 64 rows of 0 to 1,023 keys of 12 heads of 64 15.4 us for
// 51 MB, where the longest row is what is waited for; one row of 1,000 keys 7.4 us, a launch and four trips to memory.
template <typename T, int HD, bool WHOLE>
__global__ __launch_bounds__(WAVE * rows_waves(HD, sizeof(T))) void scaled_rows_attention_kernel(AttendArguments a, int run_tiles, int n_runs, float* __restrict__ parts) {
    extern __shared__ float meeting[];
    attend_row<T, HD, WHOLE>(a, blockIdx.x, blockIdx.y, blockIdx.z, blockDim.x / WAVE, run_tiles, n_runs, parts, meeting);
}

// Puts the runs of a row's head together: a wave a (row, head), four to a block; eight runs' sums are on their way at a time (5.2 us for 512 heads of four
// runs: a launch and two trips to memory).
template <typename T>
__global__ __launch_bounds__(256) void scaled_merge_kernel(AttendArguments a, int run_tiles, int n_runs, const float* __restrict__ parts) {
    constexpr bool WIDE = sizeof(T) == 4;
    extern __shared__ float factors[];   // [wave][n_runs]
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int row = blockIdx.x, head = blockIdx.y * 4 + wave, head_size = a.planes.head_size;
    if (head >= a.n_heads) return;
    const RowView view(a, row);
    if (!view.sees()) return;
    const TileRange range(view.first, view.position, a.keep);
    const int runs = runs_of(range.count, run_tiles, n_runs);
    if (runs == 1) return;
    const int pitch = head_size + 2;
    const float* const mine = parts + ((size_t)row * a.n_heads + head) * n_runs * pitch;
    float* const factor = factors + wave * n_runs;
    const float sink = sink_score(a, head);
    float top = sink;
    for (int r = lane; r < runs; r += WAVE) top = fmaxf(top, mine[r * pitch + head_size]);
    top = wave_max_total(top);
    float total = 0.0f;
    for (int r = lane; r < runs; r += WAVE) {
        const float f = weight_of<WIDE>(mine[r * pitch + head_size] - top);
        factor[r] = f;
        total += mine[r * pitch + head_size + 1] * f;
    }
    total = wave_total(total);
    if (a.sinks) total += weight_of<WIDE>(sink - top);
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");   // (the wave's own factors, by its other lanes)
    __builtin_amdgcn_wave_barrier();
    for (int d = lane; d < head_size; d += WAVE) {
        float value = 0.0f;
        for (int r0 = 0; r0 < runs; r0 += 8) {
            float part[8];
#pragma unroll
            for (int u = 0; u < 8; u++) part[u] = mine[min(r0 + u, runs - 1) * pitch + d];
#pragma unroll
            for (int u = 0; u < 8; u++) value += r0 + u < runs ? part[u] * factor[min(r0 + u, runs - 1)] : 0.0f;
        }
        put_result<T>(a, row, head * head_size + d, value / total);
    }
}

}  // namespace

int scaled_merge(const AttendArguments& a, int dtype, int n_rows, int run_tiles, int n_runs, const float* parts, hipStream_t stream) {
    mllm_count_kernel(MLLM_K_SCALED_ATTENTION_MERGE);
    const dim3 grid(n_rows, ceil_div(a.n_heads, 4));
    const size_t lds = (size_t)4 * n_runs * sizeof(float);
    if (dtype == MLLM_F32) scaled_merge_kernel<float><<<grid, 4 * WAVE, lds, stream>>>(a, run_tiles, n_runs, parts);
    else scaled_merge_kernel<bf16_t><<<grid, 4 * WAVE, lds, stream>>>(a, run_tiles, n_runs, parts);
    return mllm_check_launch("scaled_attention_merge");
}

// Rows by themselves. The keys of a row are cut into as many runs as have at most run_tiles tiles of 64 each, n_runs at most (a longer
// sequence has longer runs, so no key is left out); n_runs > 1 needs `parts`, n_rows * n_heads * n_runs * (head_size + 2) floats.
MLLM_API int mllm_scaled_attention_rows(const void* q, long long q_stride, const void* k_codes, const float* k_scales, const void* v_codes, const float* v_scales, void* out,
                                        long long out_stride, const int* token_request, const int* positions, const int* block_tables, int max_blocks, int n_tables,
                                        int num_pages, int n_rows, int n_heads, int n_kv_heads, int head_size, int page_size, int window, float scale, int dtype,
                                        float softcap, const float* sinks, int chunk, int keep, int wide_out, int out_packed, int waves, int run_tiles, int n_runs, float* parts,
                                        hipStream_t stream) {
    AttendArguments a = attend_arguments(q, q_stride, k_codes, k_scales, v_codes, v_scales, out, out_stride, block_tables, max_blocks, n_tables, num_pages, n_rows, n_heads,
                                         n_kv_heads, head_size, page_size, window, scale, dtype, softcap, sinks, chunk, keep, wide_out);
    a.token_request = token_request, a.positions = positions, a.out_packed = out_packed;
    if (int status = refuse_attend("scaled_attention_rows", a, page_size, dtype)) return status;
    const int padded = head_size <= 64 ? 64 : head_size <= 128 ? 128 : 256, most = rows_waves(padded, dtype == MLLM_F32 ? 4 : 2);
    MLLM_REQUIRE(waves >= 1 && waves <= most && run_tiles >= 1 && n_runs >= 1 && n_runs <= MOST_RUNS && (n_runs == 1 || parts != nullptr),
                 "scaled_attention_rows: %d waves (1..%d), runs of %d tiles, %d runs (with memory for more than one)", waves, most, run_tiles, n_runs);
    const int group = n_heads / n_kv_heads, columns = group < 16 ? group : 16;
    const size_t lds = (size_t)waves * columns * (head_size + 4) * sizeof(float);
    MLLM_REQUIRE(lds <= 65536, "scaled_attention_rows: %d waves of %d heads need more LDS than a block has", waves, columns);
    if (n_rows == 0) return 0;
    const dim3 grid(n_rows, n_kv_heads * ceil_div(group, 16), n_runs);
    MLLM_REQUIRE(grid.y <= 65535, "scaled_attention_rows: too many heads for one launch");
    mllm_count_kernel(MLLM_K_SCALED_ATTENTION_ROWS);
#define ROWS_LAUNCH(T, HD)                                                                                                         \
    if (page_size >= TILE_KEYS) scaled_rows_attention_kernel<T, HD, true><<<grid, waves * WAVE, lds, stream>>>(a, run_tiles, n_runs, parts); \
    else scaled_rows_attention_kernel<T, HD, false><<<grid, waves * WAVE, lds, stream>>>(a, run_tiles, n_runs, parts);
#define ROWS_CASE(T)                          \
    if (padded == 64) { ROWS_LAUNCH(T, 64) }  \
    else if (padded == 128) { ROWS_LAUNCH(T, 128) } \
    else { ROWS_LAUNCH(T, 256) }
    if (dtype == MLLM_F32) {
        ROWS_CASE(float)
    } else {
        ROWS_CASE(bf16_t)
    }
#undef ROWS_CASE
#undef ROWS_LAUNCH
    if (int status = mllm_check_launch("scaled_attention_rows")) return status;
    return n_runs == 1 ? 0 : scaled_merge(a, dtype, n_rows, run_tiles, n_runs, parts, stream);
}
