// The row-wise work between a layer's input product and its attention over a cache of 8 bits (scaled_blocks.h): queries and keys normed
// and turned by their positions, keys and values put into their blocks; and what a cache holds, read back.
#include "scaled_blocks.h"

namespace {

// What is done to the heads of one kind on their way.
struct Turn {
    const double* frequencies;   // null: nothing is turned
    int dims;                    // the first so many elements are, in pairs
    int neighbours;              // 0: elements i and i + dims / 2 are a pair; 1: 2i and 2i + 1
};

struct AppendArguments {
    const void* rows;
    long long stride;
    int q_at, k_at, v_at;                   // first columns; negative: no queries, no keys and values
    const float* q_gain;                    // null: as they are (or, with `unit`, normed without a gain)
    const float* k_gain;
    float eps;
    int unit;
    Turn turn, v_turn;
    const int* positions;
    const int* slots;
    void* q_out;
    uint8_t* k_codes;
    float* k_scales;
    uint8_t* v_codes;
    float* v_scales;
    long long n_slots;
    int n_rows, n_heads, n_kv_heads, dim, vdim, head_size, page_shift;
};

// cos and sin of position x frequency to the last bits of 64: the turns are taken off in quarters, and what is left, at most pi / 4, goes
// through the series of both (the first term left out is below 1e-16). Keys are rounded to 8 bits once, from 64: a key that lies
// next to a border falls on the side where the exact one does.
__device__ __forceinline__ void turn_of(int position, double frequency, double& c, double& s) {
    const double angle = (double)position * frequency;
    const double quarters = rint(angle * 0.63661977236758134308);
    const double x = fma(quarters, -6.123233995736766e-17, fma(quarters, -1.5707963267948966, angle));   // pi / 2 in two pieces
    const double y = x * x;
    const double sx = x * (1.0 + y * (-1.0 / 6 + y * (1.0 / 120 + y * (-1.0 / 5040 + y * (1.0 / 362880 + y * (-1.0 / 39916800 + y * (1.0 / 6227020800.0 + y * (-1.0 / 1307674368000.0))))))));
    const double cx = 1.0 + y * (-0.5 + y * (1.0 / 24 + y * (-1.0 / 720 + y * (1.0 / 40320 + y * (-1.0 / 3628800 + y * (1.0 / 479001600.0 + y * (-1.0 / 87178291200.0 + y * (1.0 / 20922789888000.0))))))));
    const int quarter = (int)((long long)quarters & 3);
    const double a = quarter & 1 ? sx : cx, b = quarter & 1 ? cx : sx;
    c = quarter == 1 || quarter == 2 ? -a : a;
    s = quarter >= 2 ? -b : b;
}

// A 64-bit number in 32 with its last bit set where anything was cut off (rounding to odd): rounded again to fewer bits it gives what the
// 64-bit number does.
__device__ __forceinline__ float sticky(double x) {
    float f = (float)x;
    const double back = (double)f;
    if (back == x || x != x) return f;
    uint32_t bits = __builtin_bit_cast(uint32_t, f);
    if (fabs(back) > fabs(x)) bits--;
    return __builtin_bit_cast(float, bits | 1u);
}

// A block: a run of rows after another (those that begin in its `per` rows), each by all its waves: the cosines and sines of the run's
// positions once for all heads, then a head's keys or values of the run at a time, or a row's query head, by a wave. A lane has
// E elements of the head, 64 apart.
template <typename T, int E>
__global__ __launch_bounds__(256) void scaled_append_kernel(AppendArguments a, int per) {
    extern __shared__ double2 turns[];   // [16][pairs] of queries and keys, then of values
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE, waves = blockDim.x / WAVE;
    const int window = blockIdx.x * per;
    const bool keeps = a.k_at >= 0;
    uint32_t begins = keeps ? run_begins(a.slots, window, a.n_rows, a.n_slots, lane) : 0xffffffffu;
    const int pairs = a.turn.frequencies ? a.turn.dims / 2 : 0, v_pairs = a.v_turn.frequencies && keeps ? a.v_turn.dims / 2 : 0;
    double2* const v_turns = turns + BLOCK_TOKENS * pairs;
    const T* rows = static_cast<const T*>(a.rows);

    while (begins) {
        const int at = __builtin_ctz(begins);
        const int first = window + at;
        if (at >= per || first >= a.n_rows) return;
        begins &= begins - 1;
        const int count = min((begins ? __builtin_ctz(begins) : 32) - at, a.n_rows - first);   // at most 16
        const int slot = keeps ? a.slots[first] : -1;
        const bool kept = slot >= 0 && slot < a.n_slots;

        for (int i = threadIdx.x; i < count * (pairs + v_pairs); i += blockDim.x) {
            const bool of_value = i >= count * pairs;
            const int j = of_value ? i - count * pairs : i, n = of_value ? v_pairs : pairs;
            double c, s;
            turn_of(a.positions[first + j / n], (of_value ? a.v_turn : a.turn).frequencies[j % n], c, s);
            (of_value ? v_turns : turns)[j] = make_double2(c, s);
        }
        __syncthreads();

        // element d of row r's head, before anything is done to it
        auto element = [&](int row, int column, int d, int size) { return d < size ? to_float(rows[(size_t)row * a.stride + column + d]) : 0.0f; };
        auto norm_factor = [&](float sum) { return rsqrtf(sum / (float)a.dim + a.eps); };
        // where the pair of element d lies, its number, and whether d is the first of the two
        auto partner = [&](const Turn& turn, int d, int& pair, bool& is_first) {
            const int half = turn.dims / 2;
            pair = turn.neighbours ? d / 2 : d % half;
            is_first = turn.neighbours ? d % 2 == 0 : d < half;
            return turn.neighbours ? d ^ 1 : is_first ? d + half : d - half;
        };

        const int jobs = kept ? 2 * a.n_kv_heads : 0;
        const int q_jobs = a.q_at >= 0 ? count * a.n_heads : 0;
        for (int job = blockIdx.y * waves + wave; job < jobs + q_jobs; job += gridDim.y * waves) {
            if (job >= jobs) {   // a row's query head
                const int row = (job - jobs) / a.n_heads, head = (job - jobs) % a.n_heads;
                const int column = a.q_at + head * a.dim;
                float x[E], factor = 1.0f;
                const bool normed = a.q_gain != nullptr || a.unit;
#pragma unroll
                for (int e = 0; e < E; e++) x[e] = element(first + row, column, lane + e * WAVE, a.dim);
                if (normed) {
                    float sum = 0.0f;
#pragma unroll
                    for (int e = 0; e < E; e++) sum += x[e] * x[e];
                    factor = norm_factor(wave_total(sum));
                }
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const int d = lane + e * WAVE;
                    auto weighted = [&](float value, int at) { return normed ? value * factor * (a.q_gain ? a.q_gain[at] : 1.0f) : value; };
                    float value = d < a.dim ? weighted(x[e], d) : 0.0f;
                    if (pairs && d < a.turn.dims) {
                        int pair;
                        bool is_first;
                        const int other = partner(a.turn, d, pair, is_first);
                        const float second = weighted(element(first + row, column, other, a.dim), other);
                        const double2 cs = turns[row * pairs + pair];
                        const float c = (float)cs.x, s = is_first ? -(float)cs.y : (float)cs.y;
                        value = value * c + second * s;
                    }
                    if (d < a.head_size) static_cast<T*>(a.q_out)[((size_t)(first + row) * a.n_heads + head) * a.head_size + d] = from_float<T>(value);
                }
                continue;
            }
            const bool of_value = job >= a.n_kv_heads;
            const int head = of_value ? job - a.n_kv_heads : job, size = of_value ? a.vdim : a.dim;
            const int column = of_value ? a.v_at + head * a.vdim : a.k_at + head * a.dim;
            const Turn& turn = of_value ? a.v_turn : a.turn;
            const int my_pairs = of_value ? v_pairs : pairs;
            const double2* my_turns = of_value ? v_turns : turns;
            const bool normed = !of_value && (a.k_gain != nullptr || a.unit);
            const int lead = slot % BLOCK_TOKENS;
            const size_t block = (((size_t)(slot >> a.page_shift) * a.n_kv_heads + head) << (a.page_shift - 4)) + ((slot & ((1 << a.page_shift) - 1)) / BLOCK_TOKENS);
            uint8_t* const codes = (of_value ? a.v_codes : a.k_codes) + block * BLOCK_TOKENS * a.head_size;
            float* const scale_at = (of_value ? a.v_scales : a.k_scales) + block;

            float x[BLOCK_TOKENS][E];
            float largest = 0.0f;
#pragma unroll
            for (int t = 0; t < BLOCK_TOKENS; t++) {
                float factor = 1.0f;
#pragma unroll
                for (int e = 0; e < E; e++) x[t][e] = t < count ? element(first + t, column, lane + e * WAVE, size) : 0.0f;
                if (normed && t < count) {
                    float sum = 0.0f;
#pragma unroll
                    for (int e = 0; e < E; e++) sum += x[t][e] * x[t][e];
                    factor = norm_factor(wave_total(sum));
                }
                auto weighted = [&](float value, int at) { return normed ? value * factor * (a.k_gain ? a.k_gain[at] : 1.0f) : value; };
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const int d = lane + e * WAVE;
                    if (t < count && d < size) {
                        float value = weighted(x[t][e], d);
                        if (my_pairs && d < turn.dims) {
                            int pair;
                            bool is_first;
                            const int other = partner(turn, d, pair, is_first);
                            const double second = weighted(element(first + t, column, other, size), other);
                            const double2 cs = my_turns[t * my_pairs + pair];
                            value = sticky(fma((double)value, cs.x, second * (is_first ? -cs.y : cs.y)));
                        }
                        x[t][e] = value;
                        largest = fmaxf(largest, counted_magnitude(value));
                    }
                }
            }
            largest = wave_max_total(largest);
            const int old = lead > 0 ? scale_exponent(*scale_at) : SCALE_LOW;
            const int exponent = max(old, needed_exponent(largest));
            const float inverse = two_to(-exponent), factor = exponent - old < 126 ? two_to(old - exponent) : 0.0f;
            const bool grown = lead > 0 && exponent > old;
            if (of_value) {
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const int d = lane + e * WAVE;
                    if (d < a.head_size) {
                        Vec16 piece = {{0u, 0u, 0u, 0u}};
                        Vec16* const at = reinterpret_cast<Vec16*>(codes + d * BLOCK_TOKENS);
                        if (count < BLOCK_TOKENS) piece = *at;
                        uint32_t fresh[4];
                        // this run's codes from token 0 on, then moved to where they belong
#pragma unroll
                        for (int w = 0; w < 4; w++)
                            fresh[w] = four_codes(ready_for_code(x[4 * w][e], inverse), ready_for_code(x[4 * w + 1][e], inverse), ready_for_code(x[4 * w + 2][e], inverse),
                                                  ready_for_code(x[4 * w + 3][e], inverse));
#pragma unroll
                        for (int w = 0; w < 4; w++) {
                            const uint32_t held = grown ? rescaled_codes(piece.w[w], factor) : piece.w[w];
                            uint32_t out = 0;
#pragma unroll
                            for (int b = 0; b < 4; b++) {
                                const int token = 4 * w + b, from = token - lead;
                                uint32_t code = token < lead ? held >> (8 * b) : piece.w[w] >> (8 * b);
                                if (from >= 0 && from < count) {
                                    const uint32_t word = from < 4 ? fresh[0] : from < 8 ? fresh[1] : from < 12 ? fresh[2] : fresh[3];
                                    code = word >> (8 * (from & 3));
                                }
                                out |= (code & 255u) << (8 * b);
                            }
                            piece.w[w] = out;
                        }
                        *at = piece;
                    }
                }
            } else {
                if (grown)
                    for (int i = lane; i < a.head_size; i += WAVE)   // (head_size / 16) x 16 pieces of 16 bytes
                        if (i % BLOCK_TOKENS < lead) {
                            Vec16* const at = reinterpret_cast<Vec16*>(codes) + i;
                            Vec16 piece = *at;
#pragma unroll
                            for (int w = 0; w < 4; w++) piece.w[w] = rescaled_codes(piece.w[w], factor);
                            *at = piece;
                        }
#pragma unroll
                for (int t = 0; t < BLOCK_TOKENS; t++)
#pragma unroll
                    for (int e = 0; e < E; e++) {
                        const int d = lane + e * WAVE;
                        if (t < count && d < a.head_size)
                            codes[((d / 16) * BLOCK_TOKENS + lead + t) * 16 + d % 16] = (uint8_t)four_codes(ready_for_code(x[t][e], inverse), 0.0f, 0.0f, 0.0f);
                    }
            }
            if (lane == 0) *scale_at = two_to(exponent);
        }
        __syncthreads();
    }
}

// What the cache holds at slots[row]: a wave per run of rows and head; slots that name no place give zeros.
template <typename T>
__global__ __launch_bounds__(256) void scaled_rows_kernel(const uint8_t* __restrict__ k_codes, const float* __restrict__ k_scales, const uint8_t* __restrict__ v_codes,
                                                          const float* __restrict__ v_scales, const int* __restrict__ slots, long long n_slots, T* __restrict__ k_out,
                                                          T* __restrict__ v_out, int n_rows, int n_kv_heads, int head_size, int page_shift) {
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
    const int window = blockIdx.x * BLOCK_TOKENS, head = blockIdx.y * 4 + wave;
    if (head >= n_kv_heads) return;
    uint32_t begins = run_begins(slots, window, n_rows, n_slots, lane);
    while (begins) {
        const int at = __builtin_ctz(begins), first = window + at;
        if (at >= BLOCK_TOKENS || first >= n_rows) return;
        begins &= begins - 1;
        const int count = min((begins ? __builtin_ctz(begins) : 32) - at, n_rows - first);
        const int slot = slots[first];
        const bool held = slot >= 0 && slot < n_slots;
        const size_t block = held ? (((size_t)(slot >> page_shift) * n_kv_heads + head) << (page_shift - 4)) + ((slot & ((1 << page_shift) - 1)) / BLOCK_TOKENS) : 0;
        const float k_scale = held ? k_scales[block] : 0.0f, v_scale = held ? v_scales[block] : 0.0f;
        const uint8_t* const k = k_codes + block * BLOCK_TOKENS * head_size;
        const uint8_t* const v = v_codes + block * BLOCK_TOKENS * head_size;
        for (int t = 0; t < count; t++) {
            const int token = held ? slots[first + t] % BLOCK_TOKENS : 0;
            const size_t to = ((size_t)(first + t) * n_kv_heads + head) * head_size;
            for (int d = lane; d < head_size; d += WAVE) {
                const float key = held ? __builtin_amdgcn_cvt_f32_fp8((int)k[((d / 16) * BLOCK_TOKENS + token) * 16 + d % 16], 0) * k_scale : 0.0f;
                const float value = held ? __builtin_amdgcn_cvt_f32_fp8((int)v[d * BLOCK_TOKENS + token], 0) * v_scale : 0.0f;
                k_out[to + d] = from_float<T>(key);
                v_out[to + d] = from_float<T>(value);
            }
        }
    }
}

int shift_of(int page_size) {
    int shift = 0;
    while ((1 << shift) < page_size) shift++;
    return shift;
}

}  // namespace

MLLM_API int mllm_scaled_append(const void* rows, long long stride, int q_at, int k_at, int v_at, const float* q_gain, const float* k_gain, float eps, int unit,
                                const double* frequencies, int rot_dims, int neighbours, const double* v_frequencies, int v_rot_dims, int v_neighbours,
                                const int* positions, const int* slots, void* q_out, void* k_codes, float* k_scales, void* v_codes, float* v_scales, int num_pages,
                                int n_rows, int n_heads, int n_kv_heads, int dim, int vdim, int head_size, int page_size, int dtype, hipStream_t stream) {
    MLLM_REQUIRE(n_rows >= 0 && n_heads > 0 && n_kv_heads > 0 && num_pages > 0, "scaled_append: bad sizes");
    MLLM_REQUIRE(head_size > 0 && head_size % 16 == 0 && head_size <= SCALED_MAX_HEAD && dim > 0 && dim <= head_size && vdim > 0 && vdim <= head_size,
                 "scaled_append: heads of %d and %d in pages for %d (a multiple of 16 up to %d)", dim, vdim, head_size, SCALED_MAX_HEAD);
    MLLM_REQUIRE(page_size >= BLOCK_TOKENS && (page_size & (page_size - 1)) == 0, "scaled_append: page size %d is no power of two of at least %d", page_size, BLOCK_TOKENS);
    MLLM_REQUIRE(dtype == MLLM_F32 || dtype == MLLM_BF16, "scaled_append: unknown dtype %d", dtype);
    MLLM_REQUIRE(q_at >= 0 || k_at >= 0, "scaled_append: neither queries nor keys");
    MLLM_REQUIRE((k_at >= 0) == (v_at >= 0), "scaled_append: keys and values are kept together");
    MLLM_REQUIRE(rot_dims >= 0 && rot_dims % 2 == 0 && rot_dims <= dim && v_rot_dims >= 0 && v_rot_dims % 2 == 0 && v_rot_dims <= vdim, "scaled_append: the rotation does not fit the heads");
    MLLM_REQUIRE((rot_dims == 0 || frequencies != nullptr) && (v_rot_dims == 0 || v_frequencies != nullptr), "scaled_append: a rotation without frequencies");
    if (n_rows == 0) return 0;   // (tensors without elements have no address)
    MLLM_REQUIRE(rows != nullptr && (q_at < 0 || q_out != nullptr) && ((rot_dims == 0 && v_rot_dims == 0) || positions != nullptr) &&
                     (k_at < 0 || (slots != nullptr && k_codes != nullptr && k_scales != nullptr && v_codes != nullptr && v_scales != nullptr)),
                 "scaled_append: a missing operand");
    AppendArguments a = {rows, stride, q_at, k_at, v_at, q_gain, k_gain, eps, unit, {rot_dims ? frequencies : nullptr, rot_dims, neighbours},
                         {v_rot_dims ? v_frequencies : nullptr, v_rot_dims, v_neighbours}, positions, slots, q_out, (uint8_t*)k_codes, k_scales, (uint8_t*)v_codes, v_scales,
                         (long long)num_pages * page_size, n_rows, n_heads, n_kv_heads, dim, vdim, head_size, shift_of(page_size)};
    const int per = n_rows >= 256 && k_at >= 0 ? BLOCK_TOKENS : 1;
    const int blocks = ceil_div(n_rows, per);
    const int jobs = (k_at >= 0 ? 2 * n_kv_heads : 0) + (q_at >= 0 ? n_heads * per : 0);
    int shares = 1;
    while (blocks * shares < 1024 && shares * 4 < jobs) shares *= 2;
    const dim3 grid(blocks, shares);
    const size_t lds = (size_t)BLOCK_TOKENS * (rot_dims / 2 + v_rot_dims / 2) * sizeof(double2);
    mllm_count_kernel(MLLM_K_SCALED_APPEND);
#define APPEND_CASE(T, E) scaled_append_kernel<T, E><<<grid, 256, lds, stream>>>(a, per)
    if (dtype == MLLM_F32) {
        if (head_size <= 64) APPEND_CASE(float, 1);
        else if (head_size <= 128) APPEND_CASE(float, 2);
        else APPEND_CASE(float, 4);
    } else {
        if (head_size <= 64) APPEND_CASE(bf16_t, 1);
        else if (head_size <= 128) APPEND_CASE(bf16_t, 2);
        else APPEND_CASE(bf16_t, 4);
    }
#undef APPEND_CASE
    return mllm_check_launch("scaled_append");
}

MLLM_API int mllm_scaled_rows(const void* k_codes, const float* k_scales, const void* v_codes, const float* v_scales, const int* slots, void* k_out, void* v_out,
                              int num_pages, int n_rows, int n_kv_heads, int head_size, int page_size, int dtype, hipStream_t stream) {
    MLLM_REQUIRE(n_rows >= 0 && n_kv_heads > 0 && num_pages > 0, "scaled_rows: bad sizes");
    MLLM_REQUIRE(head_size > 0 && head_size % 16 == 0 && head_size <= SCALED_MAX_HEAD, "scaled_rows: heads of %d (a multiple of 16 up to %d)", head_size, SCALED_MAX_HEAD);
    MLLM_REQUIRE(page_size >= BLOCK_TOKENS && (page_size & (page_size - 1)) == 0, "scaled_rows: page size %d is no power of two of at least %d", page_size, BLOCK_TOKENS);
    MLLM_REQUIRE(dtype == MLLM_F32 || dtype == MLLM_BF16, "scaled_rows: unknown dtype %d", dtype);
    if (n_rows == 0) return 0;
    const dim3 grid(ceil_div(n_rows, BLOCK_TOKENS), ceil_div(n_kv_heads, 4));
    const long long n_slots = (long long)num_pages * page_size;
    mllm_count_kernel(MLLM_K_SCALED_ROWS);
    if (dtype == MLLM_F32)
        scaled_rows_kernel<float><<<grid, 256, 0, stream>>>((const uint8_t*)k_codes, k_scales, (const uint8_t*)v_codes, v_scales, slots, n_slots, (float*)k_out, (float*)v_out,
                                                            n_rows, n_kv_heads, head_size, shift_of(page_size));
    else
        scaled_rows_kernel<bf16_t><<<grid, 256, 0, stream>>>((const uint8_t*)k_codes, k_scales, (const uint8_t*)v_codes, v_scales, slots, n_slots, (bf16_t*)k_out, (bf16_t*)v_out,
                                                             n_rows, n_kv_heads, head_size, shift_of(page_size));
    return mllm_check_launch("scaled_rows");
}
