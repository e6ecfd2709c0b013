// Attention over a cache of 8 bits (scaled_blocks.h, scaled_sweep.h).
//
// A token at position p attends to the keys max(0, p - window + 1) .. p of its request (window 0: all; with kept first keys also to those;
// or, with chunks, to the keys of its own chunk up to p). A row without a request, or at a position before the first, sees nothing:
// zeros.
#include "scaled_sweep.h"

namespace {

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

constexpr int MOST_RUNS = 1024;   // of a row: their factors lie in LDS when they are put together

// The most waves a block of rows may have: as many as have the registers they need.
constexpr int rows_waves(int padded, int size) { return padded == 64 ? (size == 2 ? 16 : 8) : 1024 / padded; }

// How many runs a row's tiles are cut into.
__device__ __forceinline__ int runs_of(int tiles, int run_tiles, int n_runs) { return min(ceil_div(tiles, run_tiles), n_runs); }

// Rows by themselves (decoding, short portions, and whatever else comes without the shape of portions): a block per row, group of up to 16
// heads that share a key/value head, and run of `run_tiles` tiles; its waves take the run's tiles in turn and meet in LDS. Rows of more
// than one run leave unnormalised sums, maximum and weight per run in `parts` ([row, head, run, head_size + 2]) for the kernel below.
// What bounds it is the cache's bytes: 2 (head_size + 0.25) a key for all heads of the group together.
template <typename T, int HD, bool WHOLE>
__global__ __launch_bounds__(WAVE * rows_waves(HD, sizeof(T))) void scaled_rows_attention_kernel(AttendArguments a, int run_tiles, int n_runs, float* __restrict__ parts) {
    constexpr bool WIDE = sizeof(T) == 4;
    typedef ScaledSweep<HD, 1, WIDE, false, WHOLE> Sweep;
    extern __shared__ float meeting[];   // [wave][column][head_size + 4]
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), waves = blockDim.x / WAVE;
    const int row = blockIdx.x, run = blockIdx.z;
    const int head_size = a.planes.head_size, group = a.n_heads / a.planes.n_kv_heads, sets = ceil_div(group, 16);
    const int kv_head = blockIdx.y / sets, head0 = kv_head * group + (blockIdx.y % sets) * 16;
    const int columns = min(16, (kv_head + 1) * group - head0);
    const RowView view(a, row);
    if (!view.sees()) {
        if (run == 0)
            for (int i = threadIdx.x; i < columns * head_size; i += blockDim.x) put_result<T>(a, row, head0 * head_size + i, 0.0f);
        return;
    }
    const TileRange range(view.first, view.position, a.keep);
    const int runs = runs_of(range.count, run_tiles, n_runs);
    if (run >= runs) return;
    const bool alone = runs == 1;
    const int share = ceil_div(range.count, runs), begin = run * share, end = min(range.count, begin + share);   // (the runs of a row are alike)

    Sweep sweep;
    sweep.init(head_size, lane);
    const int column = lane % 16;
    sweep.template load_query<T>(0, column < columns ? static_cast<const T*>(a.q) + (size_t)row * a.q_stride + (head0 + column) * head_size : nullptr, head_size, a.aligned, a.negative, lane);
    const Columns heads = {view.position, view.position, a.window, a.chunk, a.keep};
    sweep.tiles(range, begin + wave, waves, end, a.block_tables + (size_t)view.request * a.max_blocks, a.planes, kv_head, a.scale, heads, view.first, view.position, lane);

    const int pitch = head_size + 4;
    const float l = sweep.weight_sum(0);
    // the maximum is the same in the four lanes of a column: it is only raised together
    float* const mine = meeting + (wave * columns + column) * pitch;
    if (column < columns) {
#pragma unroll
        for (int dt = 0; dt < Sweep::DT; dt++)
            if (dt * 16 < head_size) *reinterpret_cast<f32x4*>(mine + dt * 16 + 4 * (lane / 16)) = sweep.o[0][dt];
        if (lane < 16) {
            mine[head_size] = sweep.m[0];
            mine[head_size + 1] = l;
        }
    }
    __syncthreads();
    // a wave without tiles has m = NO_SCORE, l = 0 and sums of 0
    for (int i = threadIdx.x; i < columns * head_size; i += blockDim.x) {
        const int c = i / head_size, d = i % head_size;
        const float* const at = meeting + c * pitch;
        float top = NO_SCORE;
        for (int w = 0; w < waves; w++) top = fmaxf(top, at[w * columns * pitch + head_size]);
        float total = 0.0f, value = 0.0f;
        for (int w = 0; w < waves; w++) {
            const float factor = weight_of<WIDE>(at[w * columns * pitch + head_size] - top);
            total += at[w * columns * pitch + head_size + 1] * factor;
            value += at[w * columns * pitch + d] * factor;
        }
        if (alone) {
            if (a.sinks) total += weight_of<WIDE>(a.sinks[head0 + c] * a.sink_factor - top);
            put_result<T>(a, row, (head0 + c) * head_size + d, value / total);
        } else {
            float* const part = parts + (((size_t)row * a.n_heads + head0 + c) * n_runs + run) * (head_size + 2);
            part[d] = value;
            if (d == 0) {
                part[head_size] = top;
                part[head_size + 1] = total;
            }
        }
    }
}

// Puts the runs of a row's head together: a wave a (row, head), four to a block; eight runs' sums are on their way at a time.
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
    float top = NO_SCORE;
    for (int r = lane; r < runs; r += WAVE) top = fmaxf(top, mine[r * pitch + head_size]);
    top = wave_max_total(top);
    float total = 0.0f;
    for (int r = lane; r < runs; r += WAVE) {
        const float f = weight_of<WIDE>(mine[r * pitch + head_size] - top);
        factor[r] = f;
        total += mine[r * pitch + head_size + 1] * f;
    }
    total = wave_total(total);
    if (a.sinks) total += weight_of<WIDE>(a.sinks[head] * a.sink_factor - top);
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
    const int context = a.context_lens[request];
    if (row0 >= q_len || context < 0 || q_first < 0) return;   // (a negative context: a padding request, whose rows are nobody's)
    const int kv_head = head / (a.n_heads / a.planes.n_kv_heads);
    const int reach = (int)min((long long)a.max_blocks << a.planes.page_shift, 2147483647LL) - 1;
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

int refuse_attend(const char* what, const AttendArguments& a, int page_size, int dtype) {
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

AttendArguments attend_arguments(const void* q, long long q_stride, const void* k_codes, const float* k_scales, const void* v_codes, const float* v_scales, void* out,
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

}  // namespace

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
    if (n_runs == 1) return 0;
    mllm_count_kernel(MLLM_K_SCALED_ATTENTION_MERGE);
    const dim3 merge_grid(n_rows, ceil_div(n_heads, 4));
    const size_t merge_lds = (size_t)4 * n_runs * sizeof(float);
    if (dtype == MLLM_F32) scaled_merge_kernel<float><<<merge_grid, 4 * WAVE, merge_lds, stream>>>(a, run_tiles, n_runs, parts);
    else scaled_merge_kernel<bf16_t><<<merge_grid, 4 * WAVE, merge_lds, stream>>>(a, run_tiles, n_runs, parts);
    return mllm_check_launch("scaled_attention_merge");
}

// Portions: the rows of request r are q_starts[r] .. q_starts[r + 1] - 1, the first of them at position context_lens[r] (negative: nobody's rows).
MLLM_API int mllm_scaled_attention_tiles(const void* q, long long q_stride, const void* k_codes, const float* k_scales, const void* v_codes, const float* v_scales, void* out,
                                         long long out_stride, const int* q_starts, const int* context_lens, const int* block_tables, int max_blocks, int n_requests,
                                         int num_pages, int n_rows, int max_q_len, int n_heads, int n_kv_heads, int head_size, int page_size, int window, float scale, int dtype,
                                         float softcap, const float* sinks, int chunk, int keep, int wide_out, hipStream_t stream) {
    AttendArguments a = attend_arguments(q, q_stride, k_codes, k_scales, v_codes, v_scales, out, out_stride, block_tables, max_blocks, n_requests, num_pages, n_rows, n_heads,
                                         n_kv_heads, head_size, page_size, window, scale, dtype, softcap, sinks, chunk, keep, wide_out);
    a.q_starts = q_starts, a.context_lens = context_lens;
    if (int status = refuse_attend("scaled_attention_tiles", a, page_size, dtype)) return status;
    MLLM_REQUIRE(n_requests <= 65535 && max_q_len <= 65535 * 16, "scaled_attention_tiles: too many requests or rows for one launch");
    if (n_rows == 0 || max_q_len <= 0) return 0;
    mllm_count_kernel(MLLM_K_SCALED_ATTENTION_TILES);
#define TILES_CASE(T, HD, CT)                                                                                   \
    {                                                                                                           \
        const dim3 grid(n_heads, ceil_div(max_q_len, 16 * CT), n_requests);                                     \
        if (page_size >= TILE_KEYS) scaled_tiles_attention_kernel<T, HD, CT, true><<<grid, 256, 0, stream>>>(a); \
        else scaled_tiles_attention_kernel<T, HD, CT, false><<<grid, 256, 0, stream>>>(a);                       \
    }
    if (dtype == MLLM_F32) {
        if (head_size <= 64) TILES_CASE(float, 64, 2)
        else if (head_size <= 128) TILES_CASE(float, 128, 1)
        else TILES_CASE(float, 256, 1)
    } else {
        if (head_size <= 64) TILES_CASE(bf16_t, 64, 4)
        else if (head_size <= 128) TILES_CASE(bf16_t, 128, 2)
        else TILES_CASE(bf16_t, 256, 1)
    }
#undef TILES_CASE
    return mllm_check_launch("scaled_attention_tiles");
}
