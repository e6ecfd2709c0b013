// Attention over a cache of 8 bits: what a row by itself takes and what a tile of a portion's rows does, for the kernels of either (scaled_attention_rows.hip,
// scaled_attention_tiles.hip) and of both at once (scaled_attention_mixed.hip); their arguments, what refuses them, and how results are written.
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

// A head's sink among its scores, in their unit and finite; no score without sinks. It counts for their maximum as well: what a sink is above all
// of them would not fit 32 bits as a weight.
__device__ __forceinline__ float sink_score(const AttendArguments& a, int head) {
    if (!a.sinks) return NO_SCORE;
    const float sink = a.sinks[head] * a.sink_factor;
    return sink > -NO_SCORE ? -NO_SCORE : sink;
}

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

// How many runs a row's tiles are cut into.
__device__ __forceinline__ int runs_of(int tiles, int run_tiles, int n_runs) { return min(ceil_div(tiles, run_tiles), n_runs); }

// A row by itself (decoding, short portions, and whatever else comes without the shape of portions), its heads of set `set` (up to 16 that share a
// key/value head), and a run of `run_tiles` tiles, by `waves` waves: they take the run's tiles in turn and meet in `meeting`
// ([wave][column][head_size + 4]). Rows of more than one run leave unnormalised sums, maximum and weight per run in `parts` ([row, head, run,
// head_size + 2]).
template <typename T, int HD, bool WHOLE>
__device__ __forceinline__ void attend_row(const AttendArguments& a, int row, int set, int run, int waves, int run_tiles, int n_runs, float* __restrict__ parts, float* meeting) {
    constexpr bool WIDE = sizeof(T) == 4;
    typedef ScaledSweep<HD, 1, WIDE, false, WHOLE> Sweep;
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), threads = waves * WAVE;
    const int head_size = a.planes.head_size, group = a.n_heads / a.planes.n_kv_heads, sets = ceil_div(group, 16);
    const int kv_head = set / sets, head0 = kv_head * group + (set % sets) * 16;
    const int columns = min(16, (kv_head + 1) * group - head0);
    const RowView view(a, row);
    if (!view.sees()) {
        if (run == 0)
            for (int i = threadIdx.x; i < columns * head_size; i += threads) put_result<T>(a, row, head0 * head_size + i, 0.0f);
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
    for (int i = threadIdx.x; i < columns * head_size; i += threads) {
        const int c = i / head_size, d = i % head_size;
        const float* const at = meeting + c * pitch;
        const float sink = alone ? sink_score(a, head0 + c) : NO_SCORE;
        float top = sink;
        for (int w = 0; w < waves; w++) top = fmaxf(top, at[w * columns * pitch + head_size]);
        float total = alone && a.sinks ? weight_of<WIDE>(sink - top) : 0.0f, value = 0.0f;
        for (int w = 0; w < waves; w++) {
            const float factor = weight_of<WIDE>(at[w * columns * pitch + head_size] - top);
            total += at[w * columns * pitch + head_size + 1] * factor;
            value += at[w * columns * pitch + d] * factor;
        }
        if (alone) put_result<T>(a, row, (head0 + c) * head_size + d, value / total);
        else {
            float* const part = parts + (((size_t)row * a.n_heads + head0 + c) * n_runs + run) * (head_size + 2);
            part[d] = value;
            if (d == 0) {
                part[head_size] = top;
                part[head_size + 1] = total;
            }
        }
    }
}

constexpr int MOST_ROWS = 65535 * 16;                   // of a portion in one launch
constexpr int MOST_REACH = 2147483647 - 2 * MOST_ROWS;   // positions, the rows of a block that a portion does not have among them, are numbers of 32 bits

// What the four waves of a block of a portion share: the queries' operands while keys are walked; then what the waves hold, row by row.
template <typename T, int HD, int CT, int SPLITS>
union TileMemory {
    bf16x8 queries[4 / SPLITS][ScaledSweep<HD, CT, sizeof(T) == 4, true, true>::Q_PIECES];
    float meeting[4][16 * CT][HD + 4];
};

// Rows of a portion: request, head and tile of 16 CT 4 / SPLITS rows. SPLITS of four waves take the tiles of keys in turn, each with statistics of
// its own, and meet in LDS; with two, the other two do the same for 16 CT rows more, at the same time, so that half of what they read comes from
// the compute unit's own cache.
template <typename T, int HD, int CT, int SPLITS, bool WHOLE>
__device__ __forceinline__ void attend_tile(const AttendArguments& a, int request, int head, int tile, TileMemory<T, HD, CT, SPLITS>& lds) {
    constexpr bool WIDE = sizeof(T) == 4;
    typedef ScaledSweep<HD, CT, WIDE, true, WHOLE> Sweep;
    constexpr int WAVES = 4, GROUPS = WAVES / SPLITS, WAVE_ROWS = 16 * CT, ROWS = GROUPS * WAVE_ROWS;
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), group = wave % GROUPS, split = wave / GROUPS;
    const int head_size = a.planes.head_size;
    const int q_first = a.q_starts[request], q_len = min(a.q_starts[request + 1], a.n_rows) - q_first;
    const int row0 = tile * ROWS;
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
    for (int i = threadIdx.x; i < ROWS * fours; i += 256) {
        const int row = i / fours, d = 4 * (i % fours);
        if (row0 + row >= q_len) break;
        const int of_group = GROUPS == 1 ? 0 : row / WAVE_ROWS, at = GROUPS == 1 ? row : row % WAVE_ROWS;
        const float sink = sink_score(a, head);
        float top = sink;
#pragma unroll
        for (int w = 0; w < SPLITS; w++) top = fmaxf(top, lds.meeting[w * GROUPS + of_group][at][HD]);
        float total = a.sinks ? weight_of<WIDE>(sink - top) : 0.0f;
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

// Puts the runs of rows together (scaled_attention_rows.hip).
int scaled_merge(const AttendArguments& a, int dtype, int n_rows, int run_tiles, int n_runs, const float* parts, hipStream_t stream);
