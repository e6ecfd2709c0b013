// One wave's pass over tiles of 64 keys (four blocks) of a cache of 8 bits (scaled_blocks.h) for up to 16 CT columns: the queries that
// share a key/value head and are looked at together (heads of a group that decode, or neighbouring rows of a prompt).
//
// S^T = K . Q^T and O^T = V^T . P^T on the 16 x 16 x 32 matrix instruction, scores and sums in 32-bit. With lane = 16 q + r:
//  * Product t of a tile takes key 16 (r / 4) + 4 t + r % 4 as its row r, so that a lane's four scores of products 0 .. 3 are those of
//    column r and all sixteen keys of block q: what it needs to be the operand of the second product (its quarter of the keys),
//    with no exchange between lanes. (The order of the keys inside a product is free as long as both operands agree.)
//  * A 16-byte load is 16 elements of one key (two quarters of a product's 32) or the 16 tokens of one value element: operands as they
//    lie in the cache, but for their conversion to bfloat16, which is exact and multiplies by the block's scale on the way
//    (v_cvt_scalef32_pk_bf16_fp8: two numbers an instruction).
//  * The running maximum of a column is raised only in a tile with a score more than 8 above it (weights up to 2^8, or e^8, in between):
//    most tiles have no exchange between lanes and no rescaling at all.
//  * Weights of a row by itself are two bfloat16 numbers, the second what the first leaves (2^-16 of the weight is lost), as over plain pages, where such rows
//    keep them in 32 bits: memory is what bounds them. In one piece they took 7.0 for 7.4 us (one row of 1,000 keys), 14.3 for 15.4 (64 of up to 1,023), and
//    as long for 16 of 20,000 and more, with results up to 32 times further off than two pieces allow before they are rounded. Weights of a portion's rows are rounded to bfloat16,
//    2^-8 of each, as over plain pages: two pieces would be half as many products again on the matrix cores that bound them, 28.0 for 20.9 us (2,048 rows,
//    12 heads of 64), 382 for 283 (8,191, 16 of 128). The sum that divides is of the weights as rounded.
// WIDE (32-bit queries and results): queries and weights go through the products as three bfloat16 pieces that add up to them exactly, so
// every product of a query or weight with a held number is exact in 32-bit.
#pragma once

#include "scaled_blocks.h"

constexpr int TILE_KEYS = 64;
constexpr float NO_SCORE = -3.0e38f;       // the running maximum before any key: finite, so that nothing seen differs from it by no number
constexpr float SCORE_SLACK = 8.0f;

// The first key a query at `position` sees: the start of its chunk, or of its window, or key 0. It never falls as the position grows.
__device__ __forceinline__ int scaled_first_key(int position, int window, int chunk) {
    if (chunk > 0) return position - position % chunk;
    return window > 0 ? max(0, position - window + 1) : 0;
}

struct ScaledPlanes {
    const uint8_t* k_codes;
    const float* k_scales;
    const uint8_t* v_codes;
    const float* v_scales;
    int num_pages, n_kv_heads, head_size, page_shift;
};

// The keys that some query of a block sees, as tiles: those of the kept first keys, then from the first key's tile to the last's.
struct TileRange {
    int kept_tiles, first_tile, count;
    int first_block, last_block, kept_blocks;   // blocks of 16 that are sure to be stored

    __device__ __forceinline__ TileRange(int first_key, int last_key, int keep) {
        keep = min(keep, first_key);
        kept_blocks = (keep + BLOCK_TOKENS - 1) / BLOCK_TOKENS;
        kept_tiles = min((keep + TILE_KEYS - 1) / TILE_KEYS, first_key / TILE_KEYS);
        first_tile = first_key / TILE_KEYS;
        first_block = first_key / BLOCK_TOKENS;
        last_block = last_key / BLOCK_TOKENS;
        count = kept_tiles + last_key / TILE_KEYS - first_tile + 1;
    }
    __device__ __forceinline__ int first_key_of(int tile) const { return (tile < kept_tiles ? tile : first_tile + tile - kept_tiles) * TILE_KEYS; }
    // a block that is sure to be stored in place of one that may not be (every key of such a one is masked)
    __device__ __forceinline__ int stored(int block) const {
        return block <= last_block && (block >= first_block || block < kept_blocks) ? block : last_block;
    }
};

// What the columns of a sweep see. Column r of group ct is the row at position min(position + 16 ct, most) (heads of one row: all at `most`); it
// sees the keys from its first (scaled_first_key) up to itself, and those below `keep`.
struct Columns {
    int position, most, window, chunk, keep;
};

struct ScoreScale {
    float factor;       // of a raw score: |scale|, times log2 e where weights are powers of two
    float cap_in, cap;  // cap > 0: score <- cap tanh(raw cap_in), cap times log2 e where weights are powers of two
};

// 2^x for scores in units of log2 e; in 32-bit e^x: with t = x log2 e as rounded and r what that leaves, 2^t (1 + r ln 2), the hardware's 2^t
// and a handful of instructions more, within two units in the last place.
template <bool WIDE>
__device__ __forceinline__ float weight_of(float x) {
    if constexpr (!WIDE) return __builtin_amdgcn_exp2f(x);
    else {
        const float t = x * 1.44269504f;
        const float r = __builtin_fmaf(x, 1.44269504f, -t) + x * 1.9259629911e-8f;   // (log2 e in two pieces)
        const float power = __builtin_amdgcn_exp2f(t);
        // (an x of minus infinity leaves no number in r, and a power of zero says what it is)
        return power > 0.0f ? __builtin_fmaf(power, r * 0.69314718f, power) : power;
    }
}

// APART: the columns are rows at positions of their own (else heads of one row, which see the same keys). WHOLE: pages of 64 tokens or more, so a
// tile lies in one page, which is looked up once by the scalar unit, and a lane's place in a tile is the same in every tile; smaller pages are
// looked up by each lane for its block.
template <int HD, int CT, bool WIDE, bool APART, bool WHOLE>
struct ScaledSweep {
    static constexpr int NC = HD / 64, DT = HD / 16, NP = WIDE ? 3 : 1;
    static constexpr int NW = WIDE ? 3 : APART ? 1 : 2;   // pieces of a weight

    // The queries' operands: rows of a portion, which all waves of a block share, in LDS ([CT][NC][2][NP][WAVE]); a row's heads in registers.
    bf16x8 q[APART ? 1 : CT][NC][2][NP];
    const bf16x8* q_shared;
    f32x4 o[CT][DT];
    f32x4 s[CT][4];
    // The running maximum and sum. In bfloat16 the weights are summed by the matrix instructions, as another row of values that are all 1 (what is
    // summed is what the values are weighted with), and every lane of a column has the whole sum; in 32-bit a lane has its own keys'.
    float m[CT], l[CT];
    f32x4 l_rows[WIDE ? 1 : CT];
    Vec16 k_raw[4][NC], v_raw[DT];
    float k_scale, v_scale;
    int k_lane[NC], v_lane, head_size;   // where a lane's pieces lie, in bytes

    __device__ __forceinline__ void init(int head_size_, int lane) {
        head_size = head_size_;
        const int quarter = lane / 16, r = lane % 16, block = BLOCK_TOKENS * head_size;
#pragma unroll
        for (int c = 0; c < NC; c++)   // (pieces beyond the head's: its last once more, which meet zeros of the query)
            k_lane[c] = min(4 * c + quarter, head_size / 16 - 1) * 256 + (r % 4) * 16 + (WHOLE ? r / 4 * block : 0);
        v_lane = r * 16 + (WHOLE ? quarter * block : 0);
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            m[ct] = NO_SCORE;
            l[ct] = 0.0f;
            if constexpr (!WIDE) l_rows[ct] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int dt = 0; dt < DT; dt++) o[ct][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }

    template <int N>
    static __device__ __forceinline__ void in_pieces(float x, bf16_t (&piece)[N]) {
        if constexpr (N < 3) {
            piece[0] = static_cast<bf16_t>(x);
            if constexpr (N == 2) piece[1] = static_cast<bf16_t>(x - to_float(piece[0]));
        } else {
            // the leading eight bits, the next eight, and the rest: cut off, not rounded, so that nothing overflows
            auto head_of = [](float y) { return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, y) & 0xffff0000u); };
            const float a = head_of(x), r = __builtin_isinf(x) ? 0.0f : x - a, b = head_of(r);
            piece[0] = static_cast<bf16_t>(a);
            piece[1] = static_cast<bf16_t>(b);
            piece[2] = static_cast<bf16_t>(r - b);
        }
    }

    // Column ct's query: `row` points at its head's first element (null: no query here). negative: a negative score scale, whose sign the queries take.
    static constexpr int Q_PIECES = CT * NC * 2 * NP * WAVE;   // of 16 bytes, in LDS
    template <typename T>
    __device__ __forceinline__ void load_query(int ct, const T* row, int head_size, bool aligned, bool negative, int lane) {
        const int quarter = lane / 16;
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int d = (4 * c + quarter) * 16 + 8 * h;
                T x[8];
                if (row != nullptr && d < head_size) {
                    if (aligned) {
#pragma unroll
                        for (int w = 0; w < (int)sizeof(T) / 2; w++) reinterpret_cast<Vec16*>(x)[w] = reinterpret_cast<const Vec16*>(row + d)[w];
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; i++) x[i] = row[d + i];
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i++) x[i] = from_float<T>(0.0f);
                }
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    bf16_t piece[NP];
                    in_pieces(negative ? -to_float(x[i]) : to_float(x[i]), piece);
#pragma unroll
                    for (int p = 0; p < NP; p++) q[APART ? 0 : ct][c][h][p][i] = piece[p];
                }
            }
    }
    __device__ __forceinline__ void share_query(int ct, bf16x8* to, int lane) {
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int p = 0; p < NP; p++) to[(((ct * NC + c) * 2 + h) * NP + p) * WAVE + lane] = q[0][c][h][p];
    }

    // Where a tile's blocks lie, as numbers of blocks: its first (WHOLE), or the lane's block of keys (r / 4) and of values (q).
    struct Places {
        long long k, v;
    };
    static __device__ __forceinline__ long long place(int block, const int* __restrict__ table, const ScaledPlanes& planes, int kv_head) {
        const int shift = planes.page_shift - 4;
        unsigned page = (unsigned)table[block >> shift];
        if constexpr (WHOLE) page = __builtin_amdgcn_readfirstlane(page);
        page = min(page, (unsigned)planes.num_pages - 1u);   // (nothing a table holds leads out of the pages)
        return (((long long)page * planes.n_kv_heads + kv_head) << shift) + (block & ((1 << shift) - 1));
    }
    static __device__ __forceinline__ Places look_up(const TileRange& range, int tile, const int* __restrict__ table, const ScaledPlanes& planes, int kv_head, int lane) {
        const int block = range.first_key_of(tile) / BLOCK_TOKENS;
        if constexpr (WHOLE) {   // (the page holds a key that is seen; what else lies in it is masked)
            const long long at = place(block, table, planes, kv_head);
            return {at, at};
        } else return {place(range.stored(block + (lane % 16) / 4), table, planes, kv_head), place(range.stored(block + lane / 16), table, planes, kv_head)};
    }

    __device__ __forceinline__ void load_keys(const Places& at, const ScaledPlanes& planes, int lane) {
        const uint8_t* const block = planes.k_codes + at.k * (BLOCK_TOKENS * head_size);
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int c = 0; c < NC; c++) k_raw[t][c] = *reinterpret_cast<const Vec16*>(block + (unsigned)k_lane[c] + 64 * t);
        k_scale = planes.k_scales[at.k + (WHOLE ? (lane % 16) / 4 : 0)];
    }
    __device__ __forceinline__ void load_values(const Places& at, const ScaledPlanes& planes, int lane) {
        const uint8_t* const block = planes.v_codes + at.v * (BLOCK_TOKENS * head_size);
        const int tiles = head_size / 16;
#pragma unroll
        for (int dt = 0; dt < DT; dt++) v_raw[dt] = *reinterpret_cast<const Vec16*>(block + (unsigned)v_lane + 256 * min(dt, tiles - 1));
        v_scale = planes.v_scales[at.v + (WHOLE ? lane / 16 : 0)];
    }

    __device__ __forceinline__ void scores(int lane) {
#pragma unroll
        for (int ct = 0; ct < CT; ct++)
#pragma unroll
            for (int t = 0; t < 4; t++) s[ct][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        // the operands of a step are converted while the matrix cores work on the step before (two conversions fit behind a product)
        constexpr int STEPS = 2 * NC;
        bf16x8 keys[2][4];
        auto convert = [&](int step) {
#pragma unroll
            for (int t = 0; t < 4; t++) keys[step % 2][t] = eight_numbers(k_raw[t][step / 2].w[2 * (step % 2)], k_raw[t][step / 2].w[2 * (step % 2) + 1], k_scale);
        };
        // .. and a query's operand is on its way from LDS for the time of two
        constexpr int AHEAD = 2, QUERIES = STEPS * CT * NP;   // number (step, ct, NP - 1 - p)
        bf16x8 ring[AHEAD + 1];
        auto query_at = [&](int n) {
            const int step = n / (CT * NP), ct = n / NP % CT, p = NP - 1 - n % NP;
            return APART ? q_shared[((ct * STEPS + step) * NP + p) * WAVE + lane] : q[APART ? 0 : ct][step / 2][step % 2][p];
        };
#pragma unroll
        for (int n = 0; n < AHEAD && n < QUERIES; n++) ring[n] = query_at(n);
        convert(0);
#pragma unroll
        for (int step = 0; step < STEPS; step++) {
            if (step + 1 < STEPS) convert(step + 1);
#pragma unroll
            for (int i = 0; i < CT * NP; i++) {
                const int n = step * CT * NP + i, ct = i / NP;
                if (n + AHEAD < QUERIES) ring[(n + AHEAD) % (AHEAD + 1)] = query_at(n + AHEAD);
#pragma unroll
                for (int t = 0; t < 4; t++) s[ct][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(keys[step % 2][t], ring[n % (AHEAD + 1)], s[ct][t], 0, 0, 0);
            }
            if constexpr (APART) {
                interleave<CT * NP, 4, 16>();
                __builtin_amdgcn_sched_barrier(0);   // (operands of all the products at once would not fit the registers)
            }
        }
    }

    // Asks the compiler for GROUPS of a read from LDS and PRODUCTS matrix instructions, with CONVERSIONS others spread among all of them.
    template <int GROUPS, int PRODUCTS, int CONVERSIONS>
    static __device__ __forceinline__ void interleave() {
        constexpr int EACH = (CONVERSIONS + GROUPS * PRODUCTS - 1) / (GROUPS * PRODUCTS);
#pragma unroll
        for (int g = 0; g < GROUPS; g++) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);    // a read from LDS
#pragma unroll
            for (int i = 0; i < PRODUCTS; i++) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);    // a matrix instruction
                __builtin_amdgcn_sched_group_barrier(0x002, EACH, 0); // others
            }
        }
    }

    // Takes the tile's scores and values into the running sums. first_key: of the tile. MASKED: some column does not see some key.
    template <bool MASKED>
    __device__ __forceinline__ void take(const ScoreScale& scale, int first_key, const Columns& columns, int lane) {
        const int key = first_key + BLOCK_TOKENS * (lane / 16);   // the lane's keys: key + 4 t + i
        uint32_t seen[CT];
        bool raise = false;
        float top[CT];
        const float factor = scale.cap > 0.0f ? 1.0f : scale.factor;   // (capped scores are in their units already)
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            if (scale.cap > 0.0f) {
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float x = s[ct][t][i] * scale.cap_in;
                        s[ct][t][i] = scale.cap * (WIDE ? tanhf(x) : 1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * 2.8853900817779268f)));
                    }
            }
            if constexpr (MASKED) {
                // bit 4 t + i: whether key + 4 t + i counts
                const int last = min(columns.position + 16 * ct, columns.most), first = scaled_first_key(last, columns.window, columns.chunk);
                auto below = [&](int end) { return (1u << min(max(end - key, 0), BLOCK_TOKENS)) - 1u; };   // keys below `end`
                seen[ct] = below(last + 1) & (~below(first) | below(columns.keep));
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float score = s[ct][t][i];   // (bits are taken of a number by itself: of a vector's element they come out as the first one's)
                        const uint32_t mask = (uint32_t)((int)(seen[ct] << (31 - 4 * t - i)) >> 31), bits = __builtin_bit_cast(uint32_t, score);
                        s[ct][t][i] = __builtin_bit_cast(float, (bits & mask) | (0xff800000u & ~mask));
                    }
            }
            float best = s[ct][0][0];
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) best = fmaxf(best, s[ct][t][i]);
            top[ct] = best * factor;
            raise |= top[ct] > m[ct] + SCORE_SLACK;
        }
        if (__any(raise)) {
#pragma unroll
            for (int ct = 0; ct < CT; ct++) {
                float best = top[ct];
                best = fmaxf(best, __shfl_xor(best, 16, WAVE));
                best = fmaxf(best, __shfl_xor(best, 32, WAVE));
                const float higher = fmaxf(m[ct], best);
                const float fall = weight_of<WIDE>(m[ct] - higher);
                m[ct] = higher;
                if constexpr (WIDE) l[ct] *= fall;
                else
#pragma unroll
                    for (int i = 0; i < 4; i++) l_rows[ct][i] *= fall;
#pragma unroll
                for (int dt = 0; dt < DT; dt++)
#pragma unroll
                    for (int i = 0; i < 4; i++) o[ct][dt][i] *= fall;
            }
        }
        bf16x8 weights[CT][2][NW];
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            float sum = 0.0f;
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float p = weight_of<WIDE>(__builtin_fmaf(s[ct][t][i], factor, -m[ct]));
                    if constexpr (WIDE) sum += p;
                    bf16_t piece[NW];
                    in_pieces(p, piece);
#pragma unroll
                    for (int n = 0; n < NW; n++) weights[ct][t / 2][n][4 * (t % 2) + i] = piece[n];
                }
            if constexpr (WIDE) l[ct] += sum;
        }
        if constexpr (!WIDE) {
            const bf16_t one = static_cast<bf16_t>(1.0f);
            const bf16x8 ones = {one, one, one, one, one, one, one, one};
#pragma unroll
            for (int ct = 0; ct < CT; ct++)
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int n = NW - 1; n >= 0; n--) l_rows[ct] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, weights[ct][h][n], l_rows[ct], 0, 0, 0);
        }
        if constexpr (MASKED) {
            // Not even a weight of zero silences a NaN: codes that are no number are taken out where no column sees them (places that nothing was
            // written to, pages that others hold) ..
            uint32_t all = 0;
#pragma unroll
            for (int ct = 0; ct < CT; ct++) all |= seen[ct];
            if constexpr (APART) {
                all |= __shfl_xor(all, 1, WAVE);
                all |= __shfl_xor(all, 2, WAVE);
                all |= __shfl_xor(all, 4, WAVE);
                all |= __shfl_xor(all, 8, WAVE);
            }
            uint32_t none = 0;
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const uint32_t bits = all >> (4 * w);   // four tokens, a byte each
                const uint32_t bytes = ((bits & 1u) | (bits & 2u) << 7 | (bits & 4u) << 14 | (bits & 8u) << 21) * 0xffu;
#pragma unroll
                for (int dt = 0; dt < DT; dt++) {
                    v_raw[dt].w[w] &= bytes;
                    if constexpr (APART) none |= not_numbers(v_raw[dt].w[w]);
                }
            }
            // .. and where some do and some do not, each goes to the columns that see it.
            if (APART && __any(none != 0)) {
#pragma unroll
                for (int dt = 0; dt < DT; dt++) {
                    Vec16 ones;
#pragma unroll
                    for (int w = 0; w < 4; w++) {
                        const uint32_t high = not_numbers(v_raw[dt].w[w]) >> 7;   // 1 in each byte that is no number
                        ones.w[w] = high * 0x38u;                                 // the code of 1
                        v_raw[dt].w[w] &= ~(high * 0xffu);
                    }
#pragma unroll
                    for (int ct = 0; ct < CT; ct++) {
                        f32x4 count = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            bf16x8 sees;
#pragma unroll
                            for (int i = 0; i < 8; i++) sees[i] = static_cast<bf16_t>((seen[ct] >> (8 * h + i)) & 1u ? 1.0f : 0.0f);
                            count = __builtin_amdgcn_mfma_f32_16x16x32_bf16(eight_numbers(ones.w[2 * h], ones.w[2 * h + 1], 1.0f), sees, count, 0, 0, 0);
                        }
#pragma unroll
                        for (int i = 0; i < 4; i++) o[ct][dt][i] = count[i] > 0.0f ? __builtin_nanf("") : o[ct][dt][i];
                        __builtin_amdgcn_sched_barrier(0);   // (a rare path: not at the price of registers)
                    }
                }
            }
        }
        bf16x8 values[2];
        auto convert = [&](int step) { values[step % 2] = eight_numbers(v_raw[step / 2].w[2 * (step % 2)], v_raw[step / 2].w[2 * (step % 2) + 1], v_scale); };
        convert(0);
#pragma unroll
        for (int step = 0; step < 2 * DT; step++) {
            if (step + 1 < 2 * DT) convert(step + 1);
#pragma unroll
            for (int ct = 0; ct < CT; ct++)
#pragma unroll
                for (int n = NW - 1; n >= 0; n--)
                    o[ct][step / 2] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(values[step % 2], weights[ct][step % 2][n], o[ct][step / 2], 0, 0, 0);
            if constexpr (APART) {
                interleave<1, CT * NW, 4>();
                if (step % 4 == 3) __builtin_amdgcn_sched_barrier(0);
            }
        }
    }

    // Tiles tile, tile + step, .. below `end`, those that all columns see whole first, then the others (the order makes no difference): all_from /
    // all_to: every column sees the keys all_from .. all_to (beside kept ones).
    __device__ __forceinline__ void tiles(const TileRange& range, int tile, int step, int end, const int* __restrict__ table, const ScaledPlanes& planes, int kv_head,
                                          const ScoreScale& scale, const Columns& columns, int all_from, int all_to, int lane) {
        // tiles whole_from .. whole_to - 1 are seen whole
        const int whole_from = max(range.kept_tiles, range.kept_tiles + ceil_div(all_from, TILE_KEYS) - range.first_tile);
        const int whole_to = min(end, range.kept_tiles + (all_to + 1) / TILE_KEYS - range.first_tile);
        const int skipped = whole_from > tile ? ceil_div(whole_from - tile, step) : 0;
        const int begin = tile + skipped * step;   // the wave's first tile that may be whole
        const int behind = begin < whole_to ? begin + ceil_div(whole_to - begin, step) * step : begin;
        some_tiles<false>(range, begin, step, whole_to, behind, behind, table, planes, kv_head, scale, columns, lane);
        some_tiles<true>(range, tile < begin ? tile : behind, step, end, begin, behind, table, planes, kv_head, scale, columns, lane);
    }

    // Tiles tile, tile + step, .. below `end`, but for those of from .. to - 1.
    template <bool MASKED>
    __device__ __forceinline__ void some_tiles(const TileRange& range, int tile, int step, int end, int from, int to, const int* __restrict__ table, const ScaledPlanes& planes, int kv_head,
                                               const ScoreScale& scale, const Columns& columns, int lane) {
        if (tile >= end) return;
        Places at = look_up(range, tile, table, planes, kv_head, lane);
        load_keys(at, planes, lane);
        load_values(at, planes, lane);
        while (tile < end) {
            const int ahead = tile + step, next = ahead >= from && ahead < to ? to : ahead;
            const bool more = next < end;
            if (more) at = look_up(range, next, table, planes, kv_head, lane);
            scores(lane);
            if (more) load_keys(at, planes, lane);   // the next tile's, while this one's weights are made
            take<MASKED>(scale, range.first_key_of(tile), columns, lane);
            if (more) load_values(at, planes, lane);
            tile = next;
        }
    }

    // The wave's sum of weights of column ct, in every lane of it.
    __device__ __forceinline__ float weight_sum(int ct) const {
        if constexpr (!WIDE) return l_rows[ct][0];
        else {
            float sum = l[ct];
            sum += __shfl_xor(sum, 16, WAVE);
            sum += __shfl_xor(sum, 32, WAVE);
            return sum;
        }
    }
};
