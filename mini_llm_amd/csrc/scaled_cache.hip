// The row-wise work between a layer's input product and its attention over a cache of 8 bits (scaled_blocks.h): queries and keys normed
// and turned by their positions, keys and values put into their blocks; and what a cache holds, read back.
#include "scaled_blocks.h"

#include <algorithm>

namespace {

// Blocks of threads that a call is shared among, if it has the heads for them: 8,192 rows of 32 + 16 heads of 128, with reading back, us with 512 / 1,024 / 1,536 / 2,048 /
// 3,072: 90 / 72 / 72 / 75 / 77 (each block makes its run's cosines again); 5,000 rows of the same in 32-bit 109 / 99 / 97 / 95 / 98.
constexpr int APPEND_BLOCKS = 1536;

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
    int n_rows, n_heads, n_kv_heads, dim, vdim, head_size, page_shift, q_wide, together;
};

// cos and sin of position x frequency to the last bits of 64: the turns are taken off in quarters, and what is left, at most pi / 4, goes
// through the series of both (the first term left out is below 1e-16). Keys and values that no norm
// has rounded are rounded to 8 bits once, from 64: a number next to a border falls on the side where the exact one does. (A norm is taken in 32 bits, and a key out of it may fall to the
// other side of a border that it lies next to: one code's step in few places.)
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
    const float f = (float)x;
    const double back = (double)f;
    const uint32_t bits = __builtin_bit_cast(uint32_t, f) - (fabs(back) > fabs(x) ? 1u : 0u);
    return __builtin_bit_cast(float, bits | (back != x ? 1u : 0u));   // (what is no number stays so)
}

// A run of rows that fall into one block, as a block of threads takes it.
struct Run {
    int first, count;      // rows first .. first + count - 1
    bool kept;             // whether they go anywhere
    int lead;              // the first one's token in its block
    size_t block_in_head;  // the block: of head 0, and how far the next head's lies
    size_t head_blocks;
};

// What becomes of a block's scale: `exponent` holds the new rows and what the block holds in front of them.
struct BlockScale {
    int exponent;
    float inverse, factor;   // of new numbers; of codes that the block holds
    bool grown;
    __device__ __forceinline__ BlockScale(float largest, int lead, float held) {
        const int old = lead > 0 ? scale_exponent(held) : SCALE_LOW;
        exponent = max(old, needed_exponent(largest));
        inverse = two_to(-exponent);
        factor = exponent - old < 126 ? two_to(old - exponent) : 0.0f;
        grown = lead > 0 && exponent > old;
    }
};

// The cosines and sines of a run's positions, [16][pitch] pairs: in 64 bits for what is rounded to 8 bits, in 32 for queries. A row is a pair longer
// than it needs to be: the lanes of a wave read the same pair of 16 rows, which would lie on the same banks.
struct TurnTable {
    const double2* wide;
    const float2* narrow;
    int pairs, pitch;   // pairs 0: nothing turns
};
__host__ __device__ __forceinline__ int turn_pitch(int pairs) { return pairs ? pairs + 1 : 0; }

// Where the pair of element d lies, its number, and whether d is the first of the two.
__device__ __forceinline__ int partner_of(const Turn& turn, int d, int& pair, bool& is_first) {
    const int half = turn.dims / 2;
    pair = turn.neighbours ? d / 2 : d % half;
    is_first = turn.neighbours ? d % 2 == 0 : d < half;
    return turn.neighbours ? d ^ 1 : is_first ? d + half : d - half;
}

// The value of a pair's element, in 64 bits and rounded once.
__device__ __forceinline__ float turned_once(float value, float other, bool is_first, double2 cs) {
    return sticky(fma((double)value, cs.x, (double)other * (is_first ? -cs.y : cs.y)));
}

// The keys that a block holds in front of the new ones, taken to its new scale: (head_size / 16) x 16 pieces of 16 bytes.
__device__ __forceinline__ void rescale_keys(uint8_t* codes, int head_size, int lead, float factor, int lane) {
    for (int i = lane; i < head_size; i += WAVE)
        if (i % BLOCK_TOKENS < lead) {
            Vec16* const at = reinterpret_cast<Vec16*>(codes) + i;
            Vec16 piece = *at;
#pragma unroll
            for (int w = 0; w < 4; w++) piece.w[w] = rescaled_codes(piece.w[w], factor);
            *at = piece;
        }
}

// A head's values of a run, by a wave: a lane has elements lane, lane + 64, .. of every row, so that what it makes of one is the 16 tokens'
// codes that lie together.
template <typename T, int E>
__device__ __forceinline__ void append_values(const AppendArguments& a, const Run& run, int head, const TurnTable& turns, int lane) {
    const size_t block = run.block_in_head + head * run.head_blocks;
    uint8_t* const codes = a.v_codes + block * BLOCK_TOKENS * a.head_size;
    const T* const from = static_cast<const T*>(a.rows) + (size_t)run.first * a.stride + a.v_at + head * a.vdim;
    const float held = a.v_scales[block];
    float x[BLOCK_TOKENS][E];
    Vec16 piece[E];
#pragma unroll
    for (int e = 0; e < E; e++) {
        const int d = lane + e * WAVE;
        const T* at = from + min(d, a.vdim - 1);   // (a row and an element that are there, whether they count or not: nothing waits for a branch)
#pragma unroll
        for (int t = 0; t < BLOCK_TOKENS; t++) {
            x[t][e] = to_float(*at);
            at += t + 1 < run.count ? a.stride : 0;
        }
#pragma unroll
        for (int t = 0; t < BLOCK_TOKENS; t++) x[t][e] = t < run.count && d < a.vdim ? x[t][e] : 0.0f;
        piece[e] = Vec16{{0u, 0u, 0u, 0u}};
        if (run.count < BLOCK_TOKENS && d < a.head_size) piece[e] = *reinterpret_cast<const Vec16*>(codes + d * BLOCK_TOKENS);
    }
    if (turns.pairs) {
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int d = lane + e * WAVE;
            if (d < a.v_turn.dims) {
                int pair;
                bool is_first;
                const int other = partner_of(a.v_turn, d, pair, is_first);
#pragma unroll
                for (int t = 0; t < BLOCK_TOKENS; t++) {
                    if (t < run.count) x[t][e] = turned_once(x[t][e], to_float(from[t * a.stride + other]), is_first, turns.wide[t * turns.pitch + pair]);
                    __builtin_amdgcn_sched_barrier(0);   // (all tokens' 64-bit numbers at once would not fit the registers)
                }
            }
        }
    }
    float largest = 0.0f;
#pragma unroll
    for (int t = 0; t < BLOCK_TOKENS; t++)
#pragma unroll
        for (int e = 0; e < E; e++) largest = fmaxf(largest, counted_magnitude(x[t][e]));
    const BlockScale scale(wave_max_total(largest), run.lead, held);
#pragma unroll
    for (int e = 0; e < E; e++) {
        const int d = lane + e * WAVE;
        uint32_t fresh[4];   // this run's codes from token 0 on, then moved to where they belong
#pragma unroll
        for (int w = 0; w < 4; w++)
            fresh[w] = four_codes(ready_for_code(x[4 * w][e], scale.inverse), ready_for_code(x[4 * w + 1][e], scale.inverse), ready_for_code(x[4 * w + 2][e], scale.inverse),
                                  ready_for_code(x[4 * w + 3][e], scale.inverse));
        if (run.count < BLOCK_TOKENS) {
            const uint64_t low = fresh[0] | (uint64_t)fresh[1] << 32, high = fresh[2] | (uint64_t)fresh[3] << 32;
            const int bits = 8 * run.lead;   // the run's codes moved up by `lead` bytes of 16
            const uint64_t up_low = bits < 64 ? low << bits : 0, up_high = bits == 0 ? high : bits < 64 ? high << bits | low >> (64 - bits) : bits == 64 ? low : low << (bits - 64);
            auto bytes_from = [](int n) { return n <= 0 ? ~0ull : n >= 8 ? 0ull : ~0ull << (8 * n); };   // bytes n .. 7
            const int end = run.lead + run.count;
            const uint64_t mine_low = bytes_from(run.lead) & ~bytes_from(end), mine_high = bytes_from(run.lead - 8) & ~bytes_from(end - 8);
            const uint64_t old_low = ~bytes_from(run.lead), old_high = ~bytes_from(run.lead - 8);
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const int shift = 32 * (w & 1);
                const uint32_t mine = (uint32_t)((w < 2 ? mine_low : mine_high) >> shift), old = (uint32_t)((w < 2 ? old_low : old_high) >> shift);
                const uint32_t moved = (uint32_t)((w < 2 ? up_low : up_high) >> shift), was = piece[e].w[w];
                const uint32_t rescaled = scale.grown ? rescaled_codes(was, scale.factor) : was;
                piece[e].w[w] = (moved & mine) | (rescaled & old) | (was & ~(mine | old));
            }
        } else {
#pragma unroll
            for (int w = 0; w < 4; w++) piece[e].w[w] = fresh[w];
        }
        if (d < a.head_size) *reinterpret_cast<Vec16*>(codes + d * BLOCK_TOKENS) = piece[e];
    }
    if (lane == 0) a.v_scales[block] = two_to(scale.exponent);
}

// A head's queries or keys of a run, by a wave, eight elements at a time: lane = 16 u + t has of row t the pieces of unit 4 e + u, two of
// eight elements each that turn with each other (or lie side by side, where nothing turns or neighbours do).
template <typename T, int E, bool KEYS>
struct HeadPieces {
    float x[E][2][8];

    // where the unit's two pieces begin
    static __device__ __forceinline__ void pieces_of(const Turn& turn, int unit, int& first, int& second) {
        const bool apart = turn.frequencies && !turn.neighbours && 16 * unit < turn.dims;
        first = apart ? 8 * unit : 16 * unit;
        second = apart ? 8 * unit + turn.dims / 2 : 16 * unit + 8;
    }

    __device__ __forceinline__ void load(const AppendArguments& a, const Run& run, int column, const float* gain, const TurnTable& turns, int lane) {
        const int token = lane % 16;
        const T* const from = static_cast<const T*>(a.rows) + (size_t)(run.first + (token < run.count ? token : 0)) * a.stride + column;
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int unit = 4 * e + lane / 16;
            int at[2];
            pieces_of(a.turn, unit, at[0], at[1]);
            const bool there = token < run.count && 16 * unit < a.dim;
#pragma unroll
            for (int p = 0; p < 2; p++) {
                Vec16 raw[sizeof(T) / 2];
#pragma unroll
                for (int w = 0; w < (int)sizeof(T) / 2; w++) raw[w] = there ? reinterpret_cast<const Vec16*>(from + at[p])[w] : Vec16{{0u, 0u, 0u, 0u}};
#pragma unroll
                for (int i = 0; i < 8; i++) x[e][p][i] = to_float(reinterpret_cast<const T*>(raw)[i]);
            }
        }
        if (gain != nullptr || a.unit) {
#pragma unroll
            for (int e = 0; e < E; e++)
#pragma unroll
                for (int p = 0; p < 2; p++)
#pragma unroll
                    for (int i = 0; i < 8; i++) sum += x[e][p][i] * x[e][p][i];
            sum += __shfl_xor(sum, 16, WAVE);   // the row's other units
            sum += __shfl_xor(sum, 32, WAVE);
            const float factor = rsqrtf(sum / (float)a.dim + a.eps);
#pragma unroll
            for (int e = 0; e < E; e++) {
                const int unit = 4 * e + lane / 16;
                int at[2];
                pieces_of(a.turn, unit, at[0], at[1]);
#pragma unroll
                for (int p = 0; p < 2; p++)
#pragma unroll
                    for (int i = 0; i < 8; i++) x[e][p][i] *= factor * (gain != nullptr && 16 * unit < a.dim ? gain[at[p] + i] : 1.0f);
            }
        }
        if (!turns.pairs) return;
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int unit = 4 * e + lane / 16;
            if (16 * unit >= a.turn.dims || token >= run.count) continue;
            const auto* const mine = table_of(turns) + token * turns.pitch;
            if (a.turn.neighbours) {
#pragma unroll
                for (int p = 0; p < 2; p++)
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        turn_pair(x[e][p][i], x[e][p][i + 1], mine[8 * unit + 4 * p + i / 2]);
                        if (KEYS && i % 4 == 2) __builtin_amdgcn_sched_barrier(0);
                    }
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    turn_pair(x[e][0][i], x[e][1][i], mine[8 * unit + i]);
                    if (KEYS && i % 2 == 1) __builtin_amdgcn_sched_barrier(0);   // (all pairs' 64-bit numbers at once would take half the registers)
                }
            }
        }
    }

    static __device__ __forceinline__ auto table_of(const TurnTable& turns) {
        if constexpr (KEYS) return turns.wide;
        else return turns.narrow;
    }
    static __device__ __forceinline__ void turn_pair(float& u, float& v, double2 cs) {
        const float a = turned_once(u, v, true, cs), b = turned_once(v, u, false, cs);
        u = a, v = b;
    }
    static __device__ __forceinline__ void turn_pair(float& u, float& v, float2 cs) {
        const float a = u * cs.x - v * cs.y, b = v * cs.x + u * cs.y;
        u = a, v = b;
    }
};

template <typename O>
__device__ __forceinline__ void store_eight(O* to, const float (&x)[8]) {
    Vec16 raw[sizeof(O) / 2];
#pragma unroll
    for (int i = 0; i < 8; i++) reinterpret_cast<O*>(raw)[i] = from_float<O>(x[i]);
#pragma unroll
    for (int w = 0; w < (int)sizeof(O) / 2; w++) reinterpret_cast<Vec16*>(to)[w] = raw[w];
}

template <typename T, int E>
__device__ __forceinline__ void queries_in_pieces(const AppendArguments& a, const Run& run, int head, const TurnTable& turns, int lane) {
    HeadPieces<T, E, false> pieces;
    pieces.load(a, run, a.q_at + head * a.dim, a.q_gain, turns, lane);
    const int token = lane % 16;
    if (token >= run.count) return;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const int unit = 4 * e + lane / 16;
        if (16 * unit >= a.head_size) continue;
        int at[2];
        pieces.pieces_of(a.turn, unit, at[0], at[1]);
        const size_t to = ((size_t)(run.first + token) * a.n_heads + head) * a.head_size;
#pragma unroll
        for (int p = 0; p < 2; p++) {
            if (a.q_wide) store_eight(static_cast<float*>(a.q_out) + to + at[p], pieces.x[e][p]);
            else store_eight(static_cast<bf16_t*>(a.q_out) + to + at[p], pieces.x[e][p]);
        }
    }
}

template <typename T, int E>
__device__ __forceinline__ void keys_in_pieces(const AppendArguments& a, const Run& run, int head, const TurnTable& turns, int lane) {
    const size_t block = run.block_in_head + head * run.head_blocks;
    uint8_t* const codes = a.k_codes + block * BLOCK_TOKENS * a.head_size;
    const float held = a.k_scales[block];
    HeadPieces<T, E, true> pieces;
    pieces.load(a, run, a.k_at + head * a.dim, a.k_gain, turns, lane);
    float largest = 0.0f;
#pragma unroll
    for (int e = 0; e < E; e++)
#pragma unroll
        for (int p = 0; p < 2; p++)
#pragma unroll
            for (int i = 0; i < 8; i++) largest = fmaxf(largest, lane % 16 < run.count ? counted_magnitude(pieces.x[e][p][i]) : 0.0f);
    const BlockScale scale(wave_max_total(largest), run.lead, held);
    if (scale.grown) rescale_keys(codes, a.head_size, run.lead, scale.factor, lane);
    const int token = lane % 16;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const int unit = 4 * e + lane / 16;
        if (16 * unit >= a.head_size || token >= run.count) continue;
        int at[2];
        pieces.pieces_of(a.turn, unit, at[0], at[1]);
#pragma unroll
        for (int p = 0; p < 2; p++) {
            float ready[8];
#pragma unroll
            for (int i = 0; i < 8; i++) ready[i] = ready_for_code(pieces.x[e][p][i], scale.inverse);
            const uint2 eight = make_uint2(four_codes(ready[0], ready[1], ready[2], ready[3]), four_codes(ready[4], ready[5], ready[6], ready[7]));
            *reinterpret_cast<uint2*>(codes + ((at[p] / 16) * BLOCK_TOKENS + run.lead + token) * 16 + at[p] % 16) = eight;
        }
    }
    if (lane == 0) a.k_scales[block] = two_to(scale.exponent);
}

// The same an element a lane, for heads and places that are no whole pieces: a row's query head ..
template <typename T, int E>
__device__ __forceinline__ void query_by_elements(const AppendArguments& a, const Run& run, int row, int head, const TurnTable& turns, int lane) {
    const T* const from = static_cast<const T*>(a.rows) + (size_t)(run.first + row) * a.stride + a.q_at + head * a.dim;
    const bool normed = a.q_gain != nullptr || a.unit;
    float x[E], factor = 1.0f, sum = 0.0f;
#pragma unroll
    for (int e = 0; e < E; e++) {
        x[e] = lane + e * WAVE < a.dim ? to_float(from[lane + e * WAVE]) : 0.0f;
        sum += x[e] * x[e];
    }
    if (normed) factor = rsqrtf(wave_total(sum) / (float)a.dim + a.eps);
    auto weighted = [&](float value, int d) { return normed ? value * (factor * (a.q_gain ? a.q_gain[d] : 1.0f)) : value; };
#pragma unroll
    for (int e = 0; e < E; e++) {
        const int d = lane + e * WAVE;
        float value = d < a.dim ? weighted(x[e], d) : 0.0f;
        if (turns.pairs && d < a.turn.dims) {
            int pair;
            bool is_first;
            const int other = partner_of(a.turn, d, pair, is_first);
            const float2 cs = turns.narrow[row * turns.pitch + pair];
            value = value * cs.x + weighted(to_float(from[other]), other) * (is_first ? -cs.y : cs.y);
        }
        const size_t to = ((size_t)(run.first + row) * a.n_heads + head) * a.head_size + d;
        if (d < a.head_size) {
            if (a.q_wide) static_cast<float*>(a.q_out)[to] = value;
            else static_cast<bf16_t*>(a.q_out)[to] = from_float<bf16_t>(value);
        }
    }
}

// .. and a head's keys of a run.
template <typename T, int E>
__device__ __forceinline__ void keys_by_elements(const AppendArguments& a, const Run& run, int head, const TurnTable& turns, int lane) {
    const size_t block = run.block_in_head + head * run.head_blocks;
    uint8_t* const codes = a.k_codes + block * BLOCK_TOKENS * a.head_size;
    const T* const from = static_cast<const T*>(a.rows) + (size_t)run.first * a.stride + a.k_at + head * a.dim;
    const bool normed = a.k_gain != nullptr || a.unit;
    const float held = a.k_scales[block];
    float x[BLOCK_TOKENS][E], largest = 0.0f;
#pragma unroll
    for (int t = 0; t < BLOCK_TOKENS; t++) {
        float factor = 1.0f, sum = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) {
            x[t][e] = t < run.count && lane + e * WAVE < a.dim ? to_float(from[t * a.stride + lane + e * WAVE]) : 0.0f;
            sum += x[t][e] * x[t][e];
        }
        if (normed && t < run.count) factor = rsqrtf(wave_total(sum) / (float)a.dim + a.eps);
        auto weighted = [&](float value, int d) { return normed ? value * (factor * (a.k_gain ? a.k_gain[d] : 1.0f)) : value; };
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int d = lane + e * WAVE;
            if (t < run.count && d < a.dim) {
                float value = weighted(x[t][e], d);
                if (turns.pairs && d < a.turn.dims) {
                    int pair;
                    bool is_first;
                    const int other = partner_of(a.turn, d, pair, is_first);
                    value = turned_once(value, weighted(to_float(from[t * a.stride + other]), other), is_first, turns.wide[t * turns.pitch + pair]);
                }
                x[t][e] = value;
                largest = fmaxf(largest, counted_magnitude(value));
            }
        }
    }
    const BlockScale scale(wave_max_total(largest), run.lead, held);
    if (scale.grown) rescale_keys(codes, a.head_size, run.lead, scale.factor, lane);
#pragma unroll
    for (int t = 0; t < BLOCK_TOKENS; t++)
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int d = lane + e * WAVE;
            if (t < run.count && d < a.head_size)
                codes[((d / 16) * BLOCK_TOKENS + run.lead + t) * 16 + d % 16] = (uint8_t)four_codes(ready_for_code(x[t][e], scale.inverse), 0.0f, 0.0f, 0.0f);
        }
    if (lane == 0) a.k_scales[block] = two_to(scale.exponent);
}

// Where a call's rows go, shared among a block's 256 threads in pieces of four that lie on 16 bytes; the first 2,048 are on their way from the start.
struct CallSlots {
    const int* from;   // the first piece
    int head, pieces, lone;
    int4 held[2];
    int lone_slot;     // a row in front of the pieces, or behind them
    __device__ __forceinline__ CallSlots(const int* __restrict__ slots, int n_rows) {
        head = min((int)(-(intptr_t)slots >> 2 & 3), n_rows);
        from = slots + head;
        pieces = (n_rows - head) / 4;
        const int thread = threadIdx.x, behind = head + 4 * pieces + thread - 4;
        lone = thread < 4 ? (thread < head ? thread : -1) : behind < n_rows ? behind : -1;
        lone_slot = slots[max(lone, 0)];
#pragma unroll
        for (int i = 0; i < 2; i++)
            if (thread + 256 * i < pieces) held[i] = reinterpret_cast<const int4*>(from)[thread + 256 * i];
    }
    // Whether the calling thread's share has a row outside first .. first + count - 1 in the block of `slot`.
    __device__ __forceinline__ bool elsewhere(int slot, int first, int count) const {
        auto counts = [&](int row, int to) { return to >> 4 == slot >> 4 && (unsigned)(row - first) >= (unsigned)count; };
        auto four = [&](int piece, int4 to) {
            const int row = head + 4 * piece;
            return counts(row, to.x) | counts(row + 1, to.y) | counts(row + 2, to.z) | counts(row + 3, to.w);
        };
        bool some = lone >= 0 && counts(lone, lone_slot);
#pragma unroll
        for (int i = 0; i < 2; i++) some |= (int)threadIdx.x + 256 * i < pieces && four(threadIdx.x + 256 * i, held[i]);
#pragma unroll 4
        for (int piece = threadIdx.x + 512; piece < pieces; piece += 256) some |= four(piece, reinterpret_cast<const int4*>(from)[piece]);
        return some;
    }
};

// Where a block's rows do not stand together, two blocks of threads would read and write its scale and rescale its codes at once: `runs_apart` finds such runs, and
// append_apart takes them.
//
// Of the runs that begin in a block of threads' rows (bits of `begins`), those whose block has rows elsewhere in the call too. A run that fills its block leaves no
// place for others, so that a prompt's are not asked. Calls of up to 256 rows are looked over by each wave. A caller whose rows stand together can say so.
template <typename Elsewhere>
__device__ __forceinline__ uint32_t runs_apart(const AppendArguments& a, uint32_t begins, int window, int per, int slot_here, bool& asked, const Elsewhere& elsewhere) {
    uint32_t apart = 0;
    while (begins) {
        const int at = __builtin_ctz(begins), first = window + at;
        if (at >= per || first >= a.n_rows) break;
        begins &= begins - 1;
        const int count = min((begins ? __builtin_ctz(begins) : 32) - at, a.n_rows - first), slot = __builtin_amdgcn_readlane(slot_here, at);
        if (count == BLOCK_TOKENS || slot < 0 || slot >= a.n_slots) continue;
        asked = true;
        apart |= __any(elsewhere(slot, first, count)) ? 1u << at : 0u;
    }
    return apart;
}

// A token of a head's keys or values, by a wave, an element a lane.
template <typename T, int E, bool KEYS>
__device__ __forceinline__ void append_token(const AppendArguments& a, int row, size_t block, int token, int head, int lane) {
    const int dim = KEYS ? a.dim : a.vdim;
    const Turn& turn = KEYS ? a.turn : a.v_turn;
    uint8_t* const codes = (KEYS ? a.k_codes : a.v_codes) + block * BLOCK_TOKENS * a.head_size;
    float* const scales = KEYS ? a.k_scales : a.v_scales;
    const T* const from = static_cast<const T*>(a.rows) + (size_t)row * a.stride + (KEYS ? a.k_at : a.v_at) + head * dim;
    const bool normed = KEYS && (a.k_gain != nullptr || a.unit);
    float x[E], sum = 0.0f, largest = 0.0f;
#pragma unroll
    for (int e = 0; e < E; e++) {
        x[e] = lane + e * WAVE < dim ? to_float(from[lane + e * WAVE]) : 0.0f;
        sum += x[e] * x[e];
    }
    const float factor = normed ? rsqrtf(wave_total(sum) / (float)dim + a.eps) : 1.0f;
    auto weighted = [&](float value, int d) { return normed ? value * (factor * (a.k_gain ? a.k_gain[d] : 1.0f)) : value; };
#pragma unroll
    for (int e = 0; e < E; e++) {
        const int d = lane + e * WAVE;
        if (d >= dim) continue;
        x[e] = weighted(x[e], d);
        if (turn.frequencies && d < turn.dims) {
            int pair;
            bool is_first;
            const int other = partner_of(turn, d, pair, is_first);
            double2 cs;
            turn_of(a.positions[row], turn.frequencies[pair], cs.x, cs.y);
            x[e] = turned_once(x[e], weighted(to_float(from[other]), other), is_first, cs);
        }
        largest = fmaxf(largest, counted_magnitude(x[e]));
    }
    const BlockScale scale(wave_max_total(largest), token, scales[block]);
    if (KEYS) {
        if (scale.grown) rescale_keys(codes, a.head_size, token, scale.factor, lane);
    } else if (scale.grown)
        for (int d = lane; d < a.head_size; d += WAVE)
            for (int t = 0; t < token; t++) codes[d * BLOCK_TOKENS + t] = (uint8_t)rescaled_codes(codes[d * BLOCK_TOKENS + t], scale.factor);
#pragma unroll
    for (int e = 0; e < E; e++) {
        const int d = lane + e * WAVE;
        if (d < a.head_size)
            codes[KEYS ? ((d / 16) * BLOCK_TOKENS + token) * 16 + d % 16 : d * BLOCK_TOKENS + token] = (uint8_t)four_codes(ready_for_code(x[e], scale.inverse), 0.0f, 0.0f, 0.0f);
    }
    if (lane == 0) scales[block] = two_to(scale.exponent);
}

// Blocks whose rows do not stand together, of the runs `apart`: who has a block's first row takes them all, one after another as their tokens are; a wave has a
// head's, first_job and every step-th from there.
template <typename T, int E>
__device__ __forceinline__ void append_apart(const AppendArguments& a, uint32_t apart, int window, int wave, int first_job, int step, int lane) {
    __shared__ int rows_of[4][BLOCK_TOKENS];   // of a block's tokens, as each wave has found them
    int* const mine = rows_of[wave];
    auto settled = [] {   // what lanes have written is read by others of their wave
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "workgroup");
        __builtin_amdgcn_wave_barrier();
    };
    while (apart) {
        const int first = window + __builtin_ctz(apart), slot = a.slots[first] & ~(BLOCK_TOKENS - 1);
        apart &= apart - 1;
        if (lane < BLOCK_TOKENS) mine[lane] = -1;
        settled();
        bool in_front = false;
#pragma unroll 8
        for (int row = lane; row < a.n_rows; row += WAVE) {
            const int to = a.slots[row];
            if ((to & ~(BLOCK_TOKENS - 1)) == slot) {
                atomicMax(&mine[to & (BLOCK_TOKENS - 1)], row);
                in_front |= row < first;
            }
        }
        settled();
        if (__any(in_front)) continue;
        const size_t block = (((size_t)(slot >> a.page_shift) * a.n_kv_heads) << (a.page_shift - 4)) + ((slot & ((1 << a.page_shift) - 1)) / BLOCK_TOKENS);
        for (int token = 0; token < BLOCK_TOKENS; token++) {
            const int row = __builtin_amdgcn_readfirstlane(mine[token]);
            if (row < 0) continue;
            for (int job = first_job; job < 2 * a.n_kv_heads; job += step) {
                const int head = job % a.n_kv_heads;
                const size_t at = block + ((size_t)head << (a.page_shift - 4));
                if (job < a.n_kv_heads) append_token<T, E, true>(a, row, at, token, head, lane);
                else append_token<T, E, false>(a, row, at, token, head, lane);
            }
            settled();
        }
    }
}

// A block of threads: a run of rows after another (those that begin in its rows: one each of the first `singles`, then `most`). The cosines and sines of the run's positions are made
// once for all heads; then every wave takes heads: keys, values, queries.
// A head of a run is one wave's, because a block has one scale: the largest magnitude is a reduction inside the wave, and what is held in front of the
// new tokens is rounded again by who knows the new scale. Few rows: bound by the chain of dependent steps (slots, positions, cosines in 64-bit, rows, the block's scale, codes) behind
// the launch, 5.2 us for one row of 12 heads of 64, 5.8 for 64 rows, 16.7 for 1,950 ragged ones (float32). Many rows: 8,192 of 32 + 16 heads of 128 (bfloat16, turned) 64 us in a row of such
// calls, 54 by itself, 185 MB (168 of rows and queries, 17 of codes) at 2.9 and 3.4 TB/s (a large copy: 4.7); vector instructions are issued in six of ten cycles, the 64-bit turns of keys among
// them, and at three waves a SIMD the rest is not hidden behind them: 168 registers do not hold one body's three kinds of heads (16 of a lane and 172 of a wave are spilled). Asking for a
// wave's next head while it works on one takes more of them: 82 us for 72 with the read-back. Looking for rows that do not stand together takes 0.3, 0.2, 0.8 and 3 us of these.
template <typename T, int E, bool PIECES>
__global__ __launch_bounds__(256, E == 1 ? 4 : E == 2 ? 3 : 1) void scaled_append_kernel(AppendArguments a, int singles, int most) {
    extern __shared__ double2 tables[];   // of queries and keys, of values, and of queries in 32 bits
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), waves = blockDim.x / WAVE;
    const bool single = (int)blockIdx.x < singles;
    const int per = single ? 1 : most, window = single ? blockIdx.x : singles + ((int)blockIdx.x - singles) * most;
    const bool keeps = a.k_at >= 0;
    uint32_t begins = per == 1 ? 0xffffffffu : 0x00010001u, apart = 0;   // (queries alone have no blocks: any rows are a run)
    int slot_here = -1;   // of row window + lane
    if (keeps) {
        bool asked = false;
        if (a.together) begins = run_begins(a.slots, window, a.n_rows, a.n_slots, lane, slot_here);
        else if (a.n_rows <= 4 * WAVE) {
            int held[4];
#pragma unroll
            for (int i = 0; i < 4; i++) held[i] = a.slots[min(lane + WAVE * i, a.n_rows - 1)];
            begins = run_begins(a.slots, window, a.n_rows, a.n_slots, lane, slot_here);
            apart = runs_apart(a, begins, window, per, slot_here, asked, [&](int slot, int first, int count) {
                bool some = false;
#pragma unroll
                for (int i = 0; i < 4; i++) some |= held[i] >> 4 == slot >> 4 && (unsigned)(min(lane + WAVE * i, a.n_rows - 1) - first) >= (unsigned)count;
                return some;
            });
        } else {
            __shared__ uint32_t met[4];
            const CallSlots call(a.slots, a.n_rows);
            begins = run_begins(a.slots, window, a.n_rows, a.n_slots, lane, slot_here);
            apart = runs_apart(a, begins, window, per, slot_here, asked, [&](int slot, int first, int count) { return call.elsewhere(slot, first, count); });
            if (asked) {
                if (lane == 0) met[wave] = apart;
                __syncthreads();
                apart = __builtin_amdgcn_readfirstlane(met[0] | met[1] | met[2] | met[3]);
            }
        }
    }
    const int pairs = a.turn.frequencies ? a.turn.dims / 2 : 0, v_pairs = a.v_turn.frequencies && keeps ? a.v_turn.dims / 2 : 0;
    double2* const wide = tables;
    double2* const v_wide = wide + BLOCK_TOKENS * turn_pitch(pairs);
    float2* const narrow = reinterpret_cast<float2*>(v_wide + BLOCK_TOKENS * turn_pitch(v_pairs));
    const TurnTable turns = {wide, narrow, pairs, turn_pitch(pairs)}, v_turns = {v_wide, nullptr, v_pairs, turn_pitch(v_pairs)};

    while (begins) {
        const int at = __builtin_ctz(begins);
        Run run;
        run.first = window + at;
        if (at >= per || run.first >= a.n_rows) break;
        begins &= begins - 1;
        run.count = __builtin_amdgcn_readfirstlane(min((begins ? __builtin_ctz(begins) : 32) - at, a.n_rows - run.first));   // at most 16
        const int slot = __builtin_amdgcn_readlane(slot_here, at);
        run.kept = slot >= 0 && slot < a.n_slots;
        run.lead = slot & (BLOCK_TOKENS - 1);
        run.head_blocks = (size_t)1 << (a.page_shift - 4);
        run.block_in_head = run.kept ? (((size_t)(slot >> a.page_shift) * a.n_kv_heads) << (a.page_shift - 4)) + ((slot & ((1 << a.page_shift) - 1)) / BLOCK_TOKENS) : 0;

        if (pairs + v_pairs) {
            for (int i = threadIdx.x; i < run.count * (pairs + v_pairs); i += blockDim.x) {
                const bool of_value = i >= run.count * pairs;
                const int j = of_value ? i - run.count * pairs : i, n = of_value ? v_pairs : pairs;
                double c, s;
                turn_of(a.positions[run.first + j / n], (of_value ? a.v_turn : a.turn).frequencies[j % n], c, s);
                const int to = (j / n) * turn_pitch(n) + j % n;
                (of_value ? v_wide : wide)[to] = make_double2(c, s);
                if (!of_value) narrow[to] = make_float2((float)c, (float)s);
            }
            __syncthreads();
        }
        const int keys = run.kept && !(apart >> at & 1) ? a.n_kv_heads : 0;
        const int queries = a.q_at < 0 ? 0 : PIECES ? a.n_heads : a.n_heads * run.count;
        for (int job = blockIdx.y * waves + wave; job < 2 * keys + queries; job += gridDim.y * waves) {
            int here = lane;
            asm volatile("" : "+s"(run.count), "+v"(here));   // (what follows from them is worked out in each job: kept across jobs it takes the registers of half the waves)
            if (job < keys) {
                if constexpr (PIECES) keys_in_pieces<T, E>(a, run, job, turns, here);
                else keys_by_elements<T, E>(a, run, job, turns, here);
            } else if (job < 2 * keys) append_values<T, E>(a, run, job - keys, v_turns, here);
            else if constexpr (PIECES) queries_in_pieces<T, E>(a, run, job - 2 * keys, turns, here);
            else query_by_elements<T, E>(a, run, (job - 2 * keys) / a.n_heads, (job - 2 * keys) % a.n_heads, turns, here);
        }
        if (pairs + v_pairs) __syncthreads();
    }
    if (apart) {
        auto again = (const __attribute__((address_space(4))) AppendArguments*)__builtin_amdgcn_kernarg_segment_ptr();
        asm volatile("" : "+s"(again));   // (the arguments read again: kept for a path that is hardly ever taken, they take the registers of the others)
        append_apart<T, E>(*(const AppendArguments*)again, apart, window, wave, blockIdx.y * 4 + wave, gridDim.y * 4, lane);
    }
}

template <typename T>
__device__ __forceinline__ void store_two(T* to, float a, float b) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float2*>(to) = make_float2(a, b);
    else *reinterpret_cast<bf16x2*>(to) = bf16x2{from_float<T>(a), from_float<T>(b)};
}

// What the cache holds at slots[row]: a wave per run of rows and head; slots that name no place give zeros. Keys: a lane takes the 16
// elements of a token that lie together. Values: the tokens of two neighbouring elements, 32 bytes; heads of at most 64 elements leave half of a
// wave, which then takes the other half of the tokens. Bound by memory where there are many rows: 8,192 of 8 heads of 128 11.4 us, 50 MB at 4.4 TB/s; one row 4.6 us.
template <typename T>
__global__ __launch_bounds__(256) void scaled_rows_kernel(const uint8_t* __restrict__ k_codes, const float* __restrict__ k_scales, const uint8_t* __restrict__ v_codes,
                                                          const float* __restrict__ v_scales, const int* __restrict__ slots, long long n_slots, T* __restrict__ k_out,
                                                          T* __restrict__ v_out, int n_rows, int n_kv_heads, int head_size, int page_shift, int per) {
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
    const int window = blockIdx.x * per, head = blockIdx.y * 4 + wave;
    if (head >= n_kv_heads) return;
    const size_t row_size = (size_t)n_kv_heads * head_size;
    int slot_here;
    uint32_t begins = run_begins(slots, window, n_rows, n_slots, lane, slot_here);
    while (begins) {
        const int at = __builtin_ctz(begins), first = window + at;
        if (at >= per || first >= n_rows) return;
        begins &= begins - 1;
        const int count = min((begins ? __builtin_ctz(begins) : 32) - at, n_rows - first);
        const int slot = __builtin_amdgcn_readlane(slot_here, at);
        T* const k_to = k_out + (size_t)first * row_size + head * head_size;
        T* const v_to = v_out + (size_t)first * row_size + head * head_size;
        if (slot < 0 || slot >= n_slots) {
            for (int t = 0; t < count; t++)
                for (int d = lane; d < head_size; d += WAVE) k_to[t * row_size + d] = v_to[t * row_size + d] = from_float<T>(0.0f);
            continue;
        }
        const int lead = slot % BLOCK_TOKENS;
        const size_t block = (((size_t)(slot >> page_shift) * n_kv_heads + head) << (page_shift - 4)) + ((slot & ((1 << page_shift) - 1)) / BLOCK_TOKENS);
        const float k_scale = k_scales[block], v_scale = v_scales[block];
        const uint8_t* const k = k_codes + block * BLOCK_TOKENS * head_size;
        const uint8_t* const v = v_codes + block * BLOCK_TOKENS * head_size;
        const int token = lane % 16 - lead;
        if (token >= 0 && token < count)
            for (int piece = lane / 16; 16 * piece < head_size; piece += 4) {
                const Vec16 codes = reinterpret_cast<const Vec16*>(k)[piece * BLOCK_TOKENS + lane % 16];
                T* const to = k_to + token * row_size + 16 * piece;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    float x[8];
#pragma unroll
                    for (int w = 0; w < 2; w++) {
                        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes.w[2 * h + w], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes.w[2 * h + w], true);
                        x[4 * w] = lo[0] * k_scale, x[4 * w + 1] = lo[1] * k_scale, x[4 * w + 2] = hi[0] * k_scale, x[4 * w + 3] = hi[1] * k_scale;
                    }
                    store_eight(to + 8 * h, x);
                }
            }
        const int shares = head_size <= 64 ? 2 : 1, share = shares == 2 ? lane / 32 : 0, words = 4 / shares;
        for (int d = 2 * (shares == 2 ? lane % 32 : lane); d < head_size; d += shares == 2 ? 64 : 128) {
            const Vec16 a = reinterpret_cast<const Vec16*>(v)[d], b = reinterpret_cast<const Vec16*>(v)[d + 1];
            T* const to = v_to + d;
#pragma unroll
            for (int w = 0; w < 4; w++) {
                if (w / words != share) continue;
                const f32x2 a_lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)a.w[w], false), a_hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)a.w[w], true);
                const f32x2 b_lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)b.w[w], false), b_hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)b.w[w], true);
                const float x[4] = {a_lo[0], a_lo[1], a_hi[0], a_hi[1]}, y[4] = {b_lo[0], b_lo[1], b_hi[0], b_hi[1]};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int t = 4 * w + i - lead;
                    if (t >= 0 && t < count) store_two(to + t * row_size, x[i] * v_scale, y[i] * v_scale);
                }
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
                                int n_rows, int n_heads, int n_kv_heads, int dim, int vdim, int head_size, int page_size, int dtype, int q_dtype, int short_rows, int together,
                                hipStream_t stream) {
    MLLM_REQUIRE(n_rows >= 0 && n_heads > 0 && n_kv_heads > 0 && num_pages > 0, "scaled_append: bad sizes");
    MLLM_REQUIRE(head_size > 0 && head_size % 16 == 0 && head_size <= SCALED_MAX_HEAD && dim > 0 && dim <= head_size && vdim > 0 && vdim <= head_size,
                 "scaled_append: heads of %d and %d in pages for %d (a multiple of 16 up to %d)", dim, vdim, head_size, SCALED_MAX_HEAD);
    MLLM_REQUIRE(page_size >= BLOCK_TOKENS && (page_size & (page_size - 1)) == 0, "scaled_append: page size %d is no power of two of at least %d", page_size, BLOCK_TOKENS);
    MLLM_REQUIRE((dtype == MLLM_F32 || dtype == MLLM_BF16) && (q_dtype == MLLM_F32 || q_dtype == MLLM_BF16), "scaled_append: unknown dtype %d or %d", dtype, q_dtype);
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
                         (long long)num_pages * page_size, n_rows, n_heads, n_kv_heads, dim, vdim, head_size, shift_of(page_size), q_dtype == MLLM_F32, together};
    // pieces of eight elements: everything lies on 16 bytes, and what turns with each other lies in whole pieces
    const int size = dtype == MLLM_F32 ? 4 : 2;
    const bool on_pieces = (uintptr_t)rows % 16 == 0 && stride * size % 16 == 0 && dim % 16 == 0 && rot_dims % 16 == 0 && (q_at < 0 || (q_at * size % 16 == 0 && (uintptr_t)q_out % 16 == 0)) &&
                           (k_at < 0 || k_at * size % 16 == 0);
    // many rows: 16 to a block of threads, which finds the runs among them; few, or those that the caller says are of many requests: a block each, so that each
    // is under way at once. 32 rows of as many requests in front of 2,016 of a prompt, keys and values of 16 heads of 64, us without / with being told: 53 / 8.8
    // (2,048 of a prompt alone 7.0); 512 single rows 34.1 / 15.5; 32 and 480 of 32 + 16 heads of 128, turned, with queries 78 / 11.9 (rows said to stand together). Queries
    // alone, 32 heads of 128 turned, us with one row / 16 a block: 32 rows 5.5 / 6.4, 64 6.0 / 6.4, 128 9.4 / 6.5, 8,192 202 / 32.6.
    const int per = n_rows >= (k_at >= 0 ? 256 : 96) ? BLOCK_TOKENS : 1;
    const int singles = per == 1 || k_at < 0 ? 0 : std::max(0, std::min(short_rows, n_rows));
    const int blocks = singles + ceil_div(n_rows - singles, per);
    const int jobs = (k_at >= 0 ? 2 * n_kv_heads : 0) + (q_at < 0 ? 0 : on_pieces ? n_heads : n_heads * per);
    const int shares = std::max(1, std::min(ceil_div(APPEND_BLOCKS, blocks), jobs / 4));
    const dim3 grid(blocks, shares);
    const size_t lds = (size_t)BLOCK_TOKENS * (turn_pitch(rot_dims / 2) * (sizeof(double2) + sizeof(float2)) + turn_pitch(v_rot_dims / 2) * sizeof(double2));
    mllm_count_kernel(MLLM_K_SCALED_APPEND);
#define APPEND_CASE(T, E)                                                              \
    if (on_pieces) scaled_append_kernel<T, E, true><<<grid, 256, lds, stream>>>(a, singles, per); \
    else scaled_append_kernel<T, E, false><<<grid, 256, lds, stream>>>(a, singles, per);
    if (dtype == MLLM_F32) {
        if (head_size <= 64) { APPEND_CASE(float, 1) }
        else if (head_size <= 128) { APPEND_CASE(float, 2) }
        else { APPEND_CASE(float, 4) }
    } else {
        if (head_size <= 64) { APPEND_CASE(bf16_t, 1) }
        else if (head_size <= 128) { APPEND_CASE(bf16_t, 2) }
        else { APPEND_CASE(bf16_t, 4) }
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
    // few rows: a block of threads for every two (most of which begin no run and have nothing to do), so that runs do not wait for each other
    const int per = (long long)n_rows * n_kv_heads >= 16384 ? BLOCK_TOKENS : 2;
    const dim3 grid(ceil_div(n_rows, per), ceil_div(n_kv_heads, 4));
    const long long n_slots = (long long)num_pages * page_size;
    mllm_count_kernel(MLLM_K_SCALED_ROWS);
    if (dtype == MLLM_F32)
        scaled_rows_kernel<float><<<grid, 256, 0, stream>>>((const uint8_t*)k_codes, k_scales, (const uint8_t*)v_codes, v_scales, slots, n_slots, (float*)k_out, (float*)v_out,
                                                            n_rows, n_kv_heads, head_size, shift_of(page_size), per);
    else
        scaled_rows_kernel<bf16_t><<<grid, 256, 0, stream>>>((const uint8_t*)k_codes, k_scales, (const uint8_t*)v_codes, v_scales, slots, n_slots, (bf16_t*)k_out, (bf16_t*)v_out,
                                                             n_rows, n_kv_heads, head_size, shift_of(page_size), per);
    return mllm_check_launch("scaled_rows");
}
