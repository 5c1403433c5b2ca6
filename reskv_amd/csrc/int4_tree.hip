// Attention of the nodes of drafted trees over a paged cache of 4-bit keys and values (include/reskv_drafts.h).
//
// Row r of a sequence and KV head is node r / G of query head r % G of the head's group; a tile has 16 rows, a wave RT
// tiles.  For 32 tokens and each of the four groups g of 32 channels, on v_mfma_f32_16x16x32_f16,
//   S_g^T [token][row] = K_g Q_g^T, codes as fp16 by masking alone (see int4.hip), and
//   S^T = low q-sum^T + sum_g scale[token, g] S_g^T,
// the first term on v_mfma_f32_16x16x16_f16 (its inner dimension is the four groups, with q-sum in three fp16 parts: see lowest), the
// others as one mixed fp32 / fp16 multiply-add per score and group, so that keys are not rounded.  The rows of the K operand are taken
// in an order of tokens that leaves lane (quarter q, row n) with the scores of the tokens 8 q .. 8 q + 7: the order in which
// V's codes lie in a lane.  Softmax and its statistics are then a lane's own but for the maximum, and the weights are the B
// operand of
//   O^T [channel][row] += V^T P^T
// as they are, without the LDS.  V = code * scale + low is rounded to fp16 once (the row that reskv_int4_gather gives; half of it where a
// scale is so large that it may pass fp16's end, twice).
//
// Scores, softmax and sums are fp32.  Weights are 2^8 exp2(x - m), m at most 6 below the row's largest score so far, rounded
// to fp16 for the product and summed as rounded: eleven bits down to 2^-22 of the largest weight.  With V and the weights rounded
// to fp16, results differ from those of 64 bits by 2.8e-4 to 2.9e-4 (1 to 64 nodes after 23 to 65001 tokens, keys with outlier channels), of
// which their own rounding is 2.07e-4; V as codes with the scales in the weights (int4.hip) would be 2.2e-4, and takes a rounding of every weight for each of the four groups instead of one.
//
// Up to 64 rows a wave works by itself on 16 or 32 of them and takes what it needs of a block from memory to registers; from
// there on four or eight waves share the operands of two blocks at a time through the LDS, where the work of making them, as
// much as that of 32 rows, is done once.  32 sequences of 4000 tokens, 32 / 8 heads, us by nodes a tree, 32 rows a wave alone / 128
// and 256 rows together, with a star as chosen: 16: 93* / 114 / 136, 20: 114 / 115* / 136, 32: 137 / 123* / 140, 48: 205 / 211 / 182*,
// 64: 246 / 217 / 187*.
//
// Bound: few rows by memory's latency and the vector ALU together (32 trees of up to 16 nodes after 2000 to 8192 tokens: 77 us and
// 10 for the merge; 370 vector instructions per block and 32 rows, the ALU issuing in half of the cycles); many rows by the vector
// ALU and the matrix cores one after the other (32 trees of 64 nodes after 8192 tokens: 370 us with the merge's 10, 745 TFLOP/s; 190 vector instructions,
// 16 of them exponentials, and 36 products per block and 32 rows: the ALU issues in 58% of the cycles, the matrix cores are busy in
// 34%, and little of that is at the same time).
// What made no difference there: the order of reads, products and sums in a wave by hand, one barrier per block or per two,
// a third buffer with the barrier before the products.  One tile of rows a wave and four waves a SIMD (registers spill) took 469 us
// where this took 434, four waves and half the rows a workgroup 468, two 580; a wave's priority while it multiplies brought 410 to
// 393, the lowest values' share in fp16 parts instead of one fp32 product 388 to 362 (the third part, and the check for values past
// fp16's end, made that 370).
#include "int4.h"
#include "reskv_drafts.h"

using namespace reskv;

namespace {

typedef _Float16 half4_t __attribute__((ext_vector_type(4)));

constexpr int kNodes = RESKV_DRAFT_NODES;
constexpr int kWavesPerSimd = 2;
constexpr int kMostWaves = 1024 * kWavesPerSimd;  // 256 CUs of 4 SIMDs
constexpr float kWeightBits = 8.0f, kSlack = 6.0f;
constexpr int kTileRows = 16;

// Work: a column is (sequence, KV head, chunk of rows), as many blocks of 32 tokens long as the sequence; the columns
// lie one behind the other and every workgroup takes an equal run of blocks.  A column that lies in one run is written
// out at once; of the others every workgroup leaves a record, of its first column at 2 w, of its last at 2 w + 1.
struct TreeArgs {
    Pool pool;
    const uint16_t* q;       // [N, Hq, 128]
    const int32_t *lengths, *offsets;
    const uint64_t* seen;    // [N] or null
    uint16_t* out;           // [N, Hq, 128]
    float* part;             // [2 groups, rows, 128]: weighted values
    float2* stat;            // [2 groups, rows]: reference of the weights, their sum
    int S, N, Hq, G, groups, max_length, max_nodes, clear_rest;
    int rows_of_chunk;
    float c;                 // scaling * log2(e)

    __device__ __forceinline__ int tokens(int s) const { return min(max(lengths[s], 0), max_length); }
    __device__ __forceinline__ int blocks(int s) const { return (tokens(s) + kBlock - 1) / kBlock; }
    __device__ __forceinline__ int nodes(int s) const { return sequence_rows(offsets, s, N).count; }  // all of them
    __device__ __forceinline__ Rows rows(int s) const {                                               // that are worked on
        const Rows r = sequence_rows(offsets, s, N);
        return {r.first, min(r.count, max_nodes)};
    }
    __device__ __forceinline__ int chunks(int s, int rows_each) const { return (rows(s).count * G + rows_each - 1) / rows_each; }
    __device__ __forceinline__ int units(int s, int rows_each) const { return blocks(s) * chunks(s, rows_each) * pool.heads; }
};

// Units (blocks of columns) of the sequences before s, and of all.
struct Sums {
    int before, all;
};
__device__ __forceinline__ Sums sum_units(const TreeArgs& A, int s, int rows_each) {
    int before = 0, all = 0;
    for (int i = lane_id(); i < A.S; i += kWave) {
        const int n = A.units(i, rows_each);
        all += n;
        before += i < s ? n : 0;
    }
    return {wave_sum_int(before), wave_sum_int(all)};
}
__device__ __forceinline__ int run_length(const TreeArgs& A, int all) { return max((all + A.groups - 1) / A.groups, 1); }

// Token of a lane's row in tile j of K: rows 4 q .. 4 q + 3 are the tokens 8 q + 4 j .. + 3.
__device__ __forceinline__ int token_of(int n, int j) { return 8 * (n >> 2) + 4 * j + (n & 3); }

// The masks of the nibbles, in vector registers: an and with an or takes one instruction then, which has no room for two
// constants.
struct Masks {
    uint32_t low, high;
    __device__ __forceinline__ Masks() : low(0x000F000Fu), high(0x00F000F0u) {
        asm("" : "+v"(low));
        asm("" : "+v"(high));
    }
};

// Eight values code * scale + low in fp16 of a dword of codes, `s` and `l` being the scales and lowest values of its
// elements: the codes become 1024 + code, or 1024 + 16 code, by masking, and code exactly from that.
__device__ __forceinline__ half8_t values_of(const Masks& M, uint32_t d, const uint4& s, const uint4& l) {
    const half2_t sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f}, back = {(_Float16)-64.0f, (_Float16)-64.0f};
    const half2_t base = {(_Float16)1024.0f, (_Float16)1024.0f};
    const uint32_t e = d >> 8, m = 0x64006400u;
    const half2_t c0 = __builtin_bit_cast(half2_t, (d & M.low) | m) - base, c2 = __builtin_bit_cast(half2_t, (e & M.low) | m) - base;
    const half2_t c1 = __builtin_elementwise_fma(__builtin_bit_cast(half2_t, (d & M.high) | m), sixteenth, back);
    const half2_t c3 = __builtin_elementwise_fma(__builtin_bit_cast(half2_t, (e & M.high) | m), sixteenth, back);
    auto h = [](uint32_t w) __attribute__((always_inline)) { return __builtin_bit_cast(half2_t, w); };
    const half2_t r0 = __builtin_elementwise_fma(c0, h(s.x), h(l.x)), r1 = __builtin_elementwise_fma(c1, h(s.y), h(l.y));
    const half2_t r2 = __builtin_elementwise_fma(c2, h(s.z), h(l.z)), r3 = __builtin_elementwise_fma(c3, h(s.w), h(l.w));
    return half8_t{r0[0], r0[1], r1[0], r1[1], r2[0], r2[1], r3[0], r3[1]};
}

// Tokens t0 and t0 + 1 of a dword: the halves of those below `valid`.
__device__ __forceinline__ uint32_t halves_below(int t0, int valid) { return (t0 < valid ? 0xFFFFu : 0u) | (t0 + 1 < valid ? 0xFFFF0000u : 0u); }
// Half of two numbers in a dword.
__device__ __forceinline__ uint32_t halves_of(uint32_t w) {
    const half2_t half = {(_Float16)0.5f, (_Float16)0.5f};
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, w) * half);
}
// The larger of each of two numbers in a dword, not negative in fp16.
__device__ __forceinline__ uint32_t pair_max(uint32_t a, uint32_t b) {
    typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(ushort2_t, a), __builtin_bit_cast(ushort2_t, b)));
}
// Scales of 2^12 and more, NaN and infinity among them: values may pass fp16's largest, by the rounding of the scale.  Half of the
// values are made then, and counted twice.
__device__ __forceinline__ bool is_odd(uint32_t scales) { return (scales & 0xFFFFu) >= 0x6C00u || scales >= 0x6C000000u; }

// The lowest value of a K scaling against the parts of a sum of q: itself for the first two, 2^-10 of it for the third.  With q's
// largest element at 2^14 and codes at 2^-24 a sum is at most 2^-4, and what its first two parts leave is up to 2^-25, fp16 numbers
// having no smaller steps there than 2^-24.  2^10 times that is rounded to 2^-25 again, and the lowest value to 2^-25 or its eleven bits:
// the share is off by at most 2^-25 of |lowest| and 2^-30, times the largest element of q, where an fp32 sum's own rounding is 2^-24 of it.
constexpr float kThird = 1024.0f;
__device__ __forceinline__ uint2 lowest(uint32_t scaling) {
    const uint32_t low = __builtin_amdgcn_perm(scaling, scaling, 0x03020302u);
    const half2_t third = {(_Float16)(1.0f / kThird), (_Float16)0.0f};
    return make_uint2(low, __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, low) * third));
}
// Two results in fp16; one past fp16's largest is that largest, as a value may be (a NaN goes on).
__device__ __forceinline__ float within(float x) { return x > 65504.0f ? 65504.0f : x < -65504.0f ? -65504.0f : x; }
__device__ __forceinline__ uint32_t pack_results(float a, float b) { return pack_halves(within(a), within(b)); }

// What a wave needs of a column, and its rows' state.
template <int RT>
struct RowState {
    half8_t q[RT][4];        // lane (row n, quarter): channels 32 g + 8 quarter + [0, 8) of each group
    half4_t sum[RT];         // sum of group `quarter`'s channels, as three fp16 numbers
    float back[RT];          // what brings the row's scores back
    uint64_t sees[RT];       // the row's nodes
    float4_t acc[RT][8];     // channels 16 ct + 4 quarter + i of row n
    float m[RT], l[RT];      // reference of the row's weights, this lane's share of their sum

    // Rows r0 .. of the sequence and KV head.  Each is brought to its own power of two, so that the sixteenth of an element,
    // which meets codes times 2^-20, keeps its bits.
    __device__ __forceinline__ void start(const TreeArgs& A, const Rows& rows, int nodes, int hk, int r0, int lane) {
        const int n = lane & 15, quarter = lane >> 4, total = rows.count * A.G;
        const uint64_t all = nodes < kNodes ? (1ull << nodes) - 1 : ~0ull;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int r = r0 + rt * kTileRows + n, node = r / A.G;
            const bool real = r < total;
            const long row = (long)(rows.first + node) * A.Hq + hk * A.G + r - node * A.G;
            float top = 0.0f, part[4];
            uint4 raw[4] = {};
            if (real) {
#pragma unroll
                for (int g = 0; g < 4; ++g) raw[g] = reinterpret_cast<const uint4*>(A.q + row * kDim)[4 * g + quarter];
            }
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const uint32_t w[4] = {raw[g].x, raw[g].y, raw[g].z, raw[g].w};
                part[g] = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float x = h2f((uint16_t)(w[e >> 1] >> (16 * (e & 1))));
                    top = fmaxf(top, fabsf(x));
                    part[g] += x;
                }
            }
            top = swap_max(top);
            const float up = top > 0.0f && top < INFINITY ? ldexpf(1.0f, 14 - ilogbf(top)) : 1.0f;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const uint32_t w[4] = {raw[g].x, raw[g].y, raw[g].z, raw[g].w};
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    q[rt][g][e] = (_Float16)(h2f((uint16_t)(w[e >> 1] >> (16 * (e & 1)))) * (e & 2 ? up * 0.0625f : up));
                part[g] = swap_sum16(part[g], part[g]);
                part[g] = swap_sum32(part[g], part[g]);
            }
            const float mine = (quarter == 0 ? part[0] : quarter == 1 ? part[1] : quarter == 2 ? part[2] : part[3]) * (up * 0x1p-24f);
            const _Float16 first = (_Float16)mine, second = (_Float16)(mine - (float)first);  // (an infinity's rest is a NaN)
            const float rest = (mine - (float)first) - (float)second;
            sum[rt] = half4_t{first, second, (_Float16)(rest * kThird), (_Float16)0.0f};
            back[rt] = A.c * (0x1p24f / up);
            sees[rt] = !real ? 0 : (A.seen ? A.seen[rows.first + node] : (2ull << node) - 1) & all;
            m[rt] = -__FLT_MAX__;
            l[rt] = 0.0f;
#pragma unroll
            for (int ct = 0; ct < 8; ++ct) acc[rt][ct] = {0.0f, 0.0f, 0.0f, 0.0f};
        }
    }

    // The weights of a block, as operands.  key(j, g): the K operand of tile j and group g; scale(g): the scales of the tokens 8
    // quarter .. + 7; low(j): lowest() of the lane's K row and group.  `valid` tokens are there, from `tree` on they
    // are nodes; `visible` gets the tokens that a row sees where some do not.  before_softmax() comes behind the scores, between(rt, i)
    // in four places among the weights of the row tile behind rt.
    template <bool SHARED, class Key, class Scale, class Low, class Before, class Between>
    __device__ __forceinline__ void weights(half8_t* p, uint32_t* visible, int valid, int tree, int quarter, Key key,
                                            Scale scale, Low low, Before before_softmax, Between between) {
        float4_t score[RT][2];
        const float4_t zero = {0.0f, 0.0f, 0.0f, 0.0f};
        if (SHARED) __builtin_amdgcn_s_setprio(1);
        half4_t lows[2];
        half8_t scales[4], keys[4][2];
        auto read = [&](int g) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < 2; ++j) keys[g][j] = key(j, g);
            scales[g] = __builtin_bit_cast(half8_t, scale(g));
        };
#pragma unroll
        for (int j = 0; j < 2; ++j) lows[j] = __builtin_bit_cast(half4_t, low(j));
        read(0);
        read(1);
        float4_t d[2][2][RT];
        auto multiply = [&](int g, int j, int rt) __attribute__((always_inline)) {
            d[g & 1][j][rt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(keys[g][j], q[rt][g], zero, 0, 0, 0);
        };
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) multiply(0, j, rt);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            if (g < 2) read(g + 2);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    if (g < 3) multiply(g + 1, j, rt);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float x = d[g & 1][j][rt][i], sc = (float)scales[g][4 * j + i];
                        score[rt][j][i] = __builtin_fmaf(x, sc, g == 0 ? 0.0f : score[rt][j][i]);  // one instruction
                    }
                    if (g == 3) score[rt][j] = __builtin_amdgcn_mfma_f32_16x16x16f16(lows[j], sum[rt], score[rt][j], 0, 0, 0);
                }
        }
        if (SHARED) __builtin_amdgcn_s_setprio(0);
        before_softmax();
        if (tree < kBlock || valid < kBlock) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                uint32_t bits = tree <= 0 ? (tree > -64 ? (uint32_t)(sees[rt] >> -tree) : 0u)
                                          : tree < kBlock ? (uint32_t)(sees[rt] << tree) | ((1u << tree) - 1u) : ~0u;
                if (valid < kBlock) bits &= (1u << valid) - 1u;
                visible[rt] = bits;
                const uint32_t mine = bits >> (8 * quarter);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (!((mine >> e) & 1u)) score[rt][e >> 2][e & 3] = -INFINITY;
            }
        }
        bool grow = false;
        float top[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            top[rt] = score[rt][0][0];
#pragma unroll
            for (int i = 1; i < 8; ++i) top[rt] = fmaxf(top[rt], score[rt][i >> 2][i & 3]);
            top[rt] *= back[rt];
            grow |= top[rt] > m[rt] + kSlack;
        }
        if (ballot(grow) != 0) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const float next = fmaxf(m[rt], swap_max(top[rt])), alpha = __builtin_amdgcn_exp2f(m[rt] - next);
                m[rt] = next;
                l[rt] *= alpha;
#pragma unroll
                for (int ct = 0; ct < 8; ++ct)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[rt][ct][i] *= alpha;
            }
        }
        const half2_t ones = {(_Float16)1.0f, (_Float16)1.0f};
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const float shift = kWeightBits - m[rt];
            float total = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                if (rt > 0) between(rt - 1, e >> 1);
                const half2_t w = {(_Float16)__builtin_amdgcn_exp2f(__builtin_fmaf(score[rt][e >> 2][e & 3], back[rt], shift)),
                                   (_Float16)__builtin_amdgcn_exp2f(__builtin_fmaf(score[rt][e >> 2][(e & 3) + 1], back[rt], shift))};
                total = __builtin_amdgcn_fdot2(w, ones, total, false);
                p[rt][e] = w[0];
                p[rt][e + 1] = w[1];
            }
            l[rt] += total;
        }
    }

    // A value tile times the weights.
    __device__ __forceinline__ void add(int ct, half8_t v, const half8_t* p) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) acc[rt][ct] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p[rt], acc[rt][ct], 0, 0, 0);
    }

    __device__ __forceinline__ void add_one(int ct, int rt, half8_t v, const half8_t* p) {
        acc[rt][ct] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p[rt], acc[rt][ct], 0, 0, 0);
    }

    // Rare: nodes whose values are no numbers (bad(g): the tokens of group g) were taken as zeros; the rows that see such a node
    // get its NaN, in the channels of its group.
    template <class Bad>
    __device__ __forceinline__ void add_bad(const uint32_t* visible, Bad bad) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                if (visible[rt] & bad(g))
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[rt][2 * g][i] = acc[rt][2 * g + 1][i] = __builtin_nanf("");
    }

    // Rows r0 .. of the chunk, to their record (of `chunk` rows) or out.
    __device__ __forceinline__ void finish(const TreeArgs& A, const Rows& rows, int hk, int r0, int in_chunk, int chunk, int record, int lane) {
        const int n = lane & 15, quarter = lane >> 4, all = rows.count * A.G;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float total = swap_sum16(l[rt], l[rt]);
            total = swap_sum32(total, total);
            const int at = in_chunk + rt * kTileRows + n, r = r0 + rt * kTileRows + n, node = r / A.G;
            if (r >= all) continue;
            if (record >= 0) {
                const long rec = (long)record * chunk + at;
                if (quarter == 0) A.stat[rec] = make_float2(m[rt], total);
                float4_t* const dst = reinterpret_cast<float4_t*>(A.part + rec * kDim) + quarter;
#pragma unroll
                for (int ct = 0; ct < 8; ++ct) dst[4 * ct] = acc[rt][ct];
            } else {
                const float inv = total == 0.0f ? 0.0f : 1.0f / total;
                uint2* const dst = reinterpret_cast<uint2*>(A.out + ((long)(rows.first + node) * A.Hq + hk * A.G + r - node * A.G) * kDim) + quarter;
#pragma unroll
                for (int ct = 0; ct < 8; ++ct)
                    dst[4 * ct] = make_uint2(pack_results(acc[rt][ct][0] * inv, acc[rt][ct][1] * inv), pack_results(acc[rt][ct][2] * inv, acc[rt][ct][3] * inv));
            }
        }
    }
};

// The blocks of a column one after the other: where they lie.  Page numbers come 64 at a time, one per lane, and a page's
// address is worked out once.
struct Walk {
    int entry0, entry, inside, numbers;
    bool there;
    const char* at;  // the next block, where there is one
    __device__ __forceinline__ void fetch(const TreeArgs& A, int s, int lane) {
        numbers = A.pool.table[(long)s * A.pool.width + min(entry0 + lane, A.pool.width - 1)];
    }
    __device__ __forceinline__ void page(const TreeArgs& A, int hk) {
        const char* const p = A.pool.in_page(__builtin_amdgcn_readlane(numbers, entry), inside, hk);
        there = p != nullptr;
        at = there ? p : A.pool.pages;
    }
    __device__ __forceinline__ void start(const TreeArgs& A, int s, int hk, int begin, int lane) {
        entry0 = begin / A.pool.blocks;
        entry = 0;
        inside = begin - entry0 * A.pool.blocks;
        fetch(A, s, lane);
        page(A, hk);
    }
    __device__ __forceinline__ void next(const TreeArgs& A, int s, int hk, int lane) {
        if (++inside < A.pool.blocks) {
            if (there) at += kBlockBytes;
            return;
        }
        inside = 0;
        if (++entry == kWave) {
            entry0 += kWave;
            entry = 0;
            fetch(A, s, lane);
        }
        page(A, hk);
    }
};

// Loads of a block whose address is the same for all lanes: a lane has its offset, so that no address is worked out.
struct BlockLoads {
    __amdgpu_buffer_rsrc_t block;
    __device__ __forceinline__ explicit BlockLoads(const char* p)
        : block(__builtin_amdgcn_make_buffer_rsrc((void*)p, 0, kBlockBytes, 0x00020000)) {}
    __device__ __forceinline__ uint4 b128(int lane, int at) const {
        return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(block, lane, at, 0));
    }
    __device__ __forceinline__ uint2 b64(int lane, int at) const {
        return __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(block, lane, at, 0));
    }
    __device__ __forceinline__ uint32_t b32(int lane, int at) const { return __builtin_amdgcn_raw_buffer_load_b32(block, lane, at, 0); }
};

// ---------------------------------------------------------------------------
// few rows: a wave by itself
// ---------------------------------------------------------------------------

// One block as a lane takes it.
struct TreeBlock {
    uint4 k[2];      // tokens token_of(j), channels 8 quarter + [0, 8) of the four groups
    uint32_t ks[2];  // their scale and low of group `quarter`
    uint4 v[2];      // channels 16 (4 i + j) + lane % 16 (dword j), tokens 8 quarter + [0, 8)
    uint32_t vs, vl; // scales and lowest values of group lane / 16, tokens 2 (lane % 16) + [0, 2)
};
__device__ __forceinline__ void load_block(TreeBlock& b, const char* p, int lane) {
    const int n = lane & 15, quarter = lane >> 4;
    const BlockLoads L(p);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int t = token_of(n, j);
        b.k[j] = L.b128(16 * ((t >> 4) * 64 + quarter * 16 + (t & 15)), 0);
        b.ks[j] = L.b32(4 * (((t >> 4) * 4 + quarter) * 16 + (t & 15)), kKScale);
    }
    b.v[0] = L.b128(16 * lane, kVCodes);
    b.v[1] = L.b128(16 * lane, kVCodes + 1024);
    b.vs = L.b32(4 * lane, kVScale);
    b.vl = L.b32(4 * lane, kVLow);
}
__device__ __forceinline__ uint32_t dword(const uint4& x, int i) { return i == 0 ? x.x : i == 1 ? x.y : i == 2 ? x.z : x.w; }

struct OneWave {  // LDS
    alignas(16) uint16_t scale[4 * kBlock];
    alignas(16) uint32_t vs[64], vl[64];
};

template <int RT>
__device__ __forceinline__ void work_alone(const TreeArgs& A, OneWave& L, int s, int column, int begin, int end, int record) {
    constexpr int kRows = RT * kTileRows;
    const int lane = threadIdx.x, n = lane & 15, quarter = lane >> 4;
    const Rows rows = A.rows(s);
    const int chunks = A.chunks(s, kRows), hk = column / chunks, r0 = (column - hk * chunks) * kRows;
    const int nodes = A.nodes(s), length = A.tokens(s), context = length - nodes;
    Walk at;
    at.start(A, s, hk, begin, lane);
    TreeBlock x0, x1;
    // Block blk; behind the last one it is loaded again: a branch around the loads would have every wait for one of them wait for
    // the next block's as well.
    auto fetch = [&](TreeBlock& x, int blk) __attribute__((always_inline)) {
        const bool there = at.there;
        load_block(x, at.at, lane);
        if (blk + 1 < end) at.next(A, s, hk, lane);
        return there;
    };
    bool there0 = fetch(x0, begin), there1;  // before Q, so that the first block does not wait for it
    RowState<RT> R;
    R.start(A, rows, nodes, hk, r0, lane);
    const Masks M;

    auto work = [&](TreeBlock& x, int blk, bool there) __attribute__((always_inline)) {
        // the two waves of a SIMD go first in turns: the older one would end long before the other, which is then alone
        if ((blk ^ (int)blockIdx.x ^ ((int)blockIdx.x >> 10)) & 2) __builtin_amdgcn_s_setprio(1);
        else __builtin_amdgcn_s_setprio(0);
        if (!there) return;  // its tokens are not there
        const int valid = min(kBlock, length - blk * kBlock), tree = context - blk * kBlock;  // tokens; where the nodes begin
        if (valid < kBlock) {  // what lies behind the last token may be anything
            const uint32_t keep = halves_below(2 * n, valid);
            x.vs &= keep;
            x.vl &= keep;
        }
        const bool odd = ballot(is_odd(x.vs)) != 0;
        uint64_t bad0 = 0, bad1 = 0;  // nodes (even and odd tokens, 16 a group) whose values are no numbers
        if (odd && tree < kBlock) {
            const bool b0 = 2 * n >= tree && (x.vs & 0xFFFFu) >= 0x7C00u, b1 = 2 * n + 1 >= tree && x.vs >= 0x7C000000u;
            bad0 = ballot(b0);
            bad1 = ballot(b1);
            const uint32_t keep = (b0 ? 0u : 0xFFFFu) | (b1 ? 0u : 0xFFFF0000u);
            x.vs &= keep;
            x.vl &= keep;
        }
        if (odd) {
            x.vs = halves_of(x.vs);
            x.vl = halves_of(x.vl);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) L.scale[quarter * kBlock + token_of(n, j)] = (uint16_t)x.ks[j];
        L.vs[lane] = x.vs;
        L.vl[lane] = x.vl;
        wave_sync();
        half8_t p[RT];
        uint32_t visible[RT];
        R.template weights<false>(p, visible, valid, tree, quarter,
                                  [&](int j, int g) __attribute__((always_inline)) { return operand(dword(x.k[j], g)); },
                                  [&](int g) __attribute__((always_inline)) { return reinterpret_cast<const uint4*>(L.scale)[4 * g + quarter]; },
                                  [&](int j) __attribute__((always_inline)) { return lowest(x.ks[j]); }, []() {}, [](int, int) {});
        auto value = [&](int ct) __attribute__((always_inline)) {
            const int of = 4 * (ct >> 1) + quarter;
            return values_of(M, dword(x.v[ct >> 2], ct & 3), reinterpret_cast<const uint4*>(L.vs)[of], reinterpret_cast<const uint4*>(L.vl)[of]);
        };
        if (odd) {
            const _Float16 two = (_Float16)2.0f;
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) p[rt] *= half8_t{two, two, two, two, two, two, two, two};
        }
#pragma unroll
        for (int ct = 0; ct < 8; ++ct) R.add(ct, value(ct), p);
        if ((bad0 | bad1) != 0)
            R.add_bad(visible, [&](int g) {
                uint32_t bits = 0;
                for (int t = 0; t < kBlock; ++t) bits |= (uint32_t)((t & 1 ? bad1 : bad0) >> (16 * g + (t >> 1)) & 1u) << t;
                return bits;
            });
        wave_sync();
    };
    for (int blk = begin; blk < end; blk += 2) {
        there1 = fetch(x1, blk + 1);
        work(x0, blk, there0);
        if (blk + 1 >= end) break;
        there0 = fetch(x0, blk + 2);
        work(x1, blk + 1, there1);
    }
    R.finish(A, rows, hk, r0, 0, kRows, record, lane);
    wave_sync();
}

// ---------------------------------------------------------------------------
// more rows: waves that share a block's operands
// ---------------------------------------------------------------------------

// A block as operands in the LDS: the codes of K as fp16 numbers, its scales and lowest values, and V in fp16.
struct Operands {
    uint4 k[2][4][kWave], v[8][kWave];
    alignas(16) uint16_t scale[4 * kBlock];
    uint2 low[4 * kBlock];
    uint32_t bad[4];  // tokens of a group whose values are no numbers, where nodes are
    int odd[4];       // groups whose values are halves, where they have the number of the step (its first block's, from 1)
    int any_odd;      // of a step's first block: that number, where the step has any
};

// A wave's share of that work: pieces of K and V.
struct Share {
    uint2 k;         // task t: tokens token_of(t / 2), groups 2 (t % 2) and the next
    uint32_t ks;     // scale and low of token `lane` of group t
    uint2 v;         // task t: channels 32 t + lane % 16 and 16 further on, tokens 8 quarter + [0, 8)
    uint4 vs, vl;    // their scales and lowest values
};

constexpr int kStep = 2;  // blocks

// WAVES waves of 32 rows each take kStep blocks per step; the blocks' four tasks each are shared out among the waves.  A block that
// is not there counts as one without tokens.
template <int WAVES>
__device__ __forceinline__ void work_together(const TreeArgs& A, Operands (*L)[kStep], int s, int column, int begin, int end, int record) {
    constexpr int RT = 2, kWaveRows = RT * kTileRows, kRows = WAVES * kWaveRows, kItems = 4 * kStep / WAVES;
    const int lane = threadIdx.x & 63, n = lane & 15, quarter = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Rows rows = A.rows(s);
    const int chunks = A.chunks(s, kRows), hk = column / chunks, r0 = (column - hk * chunks) * kRows + wave * kWaveRows;
    const int nodes = A.nodes(s), length = A.tokens(s), context = length - nodes;
    const bool active = r0 < rows.count * A.G;
    Walk at;
    at.start(A, s, hk, begin, lane);
    Share x[kItems];
    // the wave's shares of the blocks blk .. blk + kStep - 1; which of them are there, as bits
    auto fetch = [&](int blk) __attribute__((always_inline)) {
        const char* found[kStep];
        uint32_t there = 0;
#pragma unroll
        for (int b = 0; b < kStep; ++b) {
            there |= (uint32_t)(at.there && blk + b < end) << b;
            found[b] = at.at;
            if (blk + b + 1 < end) at.next(A, s, hk, lane);
        }
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
            const int item = wave + i * WAVES, task = item & 3, t = token_of(n, task >> 1), u = lane & 31;
            const char* const p = item < 4 ? found[0] : found[1];
            const BlockLoads P(p);
            x[i].k = P.b64(16 * ((t >> 4) * 64 + quarter * 16 + (t & 15)) + 8 * (task & 1), 0);
            x[i].ks = P.b32(4 * (((u >> 4) * 4 + task) * 16 + (u & 15)), kKScale);
            x[i].v = P.b64(16 * ((task >> 1) * 64 + lane) + 8 * (task & 1), kVCodes);
            x[i].vs = P.b128(16 * (task * 4 + quarter), kVScale);
            x[i].vl = P.b128(16 * (task * 4 + quarter), kVLow);
        }
        return there;
    };
    auto valid_of = [&](int blk, bool there) { return there ? min(kBlock, length - blk * kBlock) : 0; };
    const Masks M;
    auto stage = [&](Operands* O0, int blk0, uint32_t there) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
            const int item = wave + i * WAVES, task = item & 3, b = item >> 2;
            Operands& O = O0[b];
            const int valid = valid_of(blk0 + b, there >> b & 1), tree = context - (blk0 + b) * kBlock;
            O.k[task >> 1][2 * (task & 1)][lane] = __builtin_bit_cast(uint4, operand(x[i].k.x));
            O.k[task >> 1][2 * (task & 1) + 1][lane] = __builtin_bit_cast(uint4, operand(x[i].k.y));
            if (lane < kBlock) {
                O.scale[task * kBlock + lane] = (uint16_t)x[i].ks;
                O.low[task * kBlock + lane] = lowest(x[i].ks);
            }
            uint32_t sc[4] = {x[i].vs.x, x[i].vs.y, x[i].vs.z, x[i].vs.w}, lo[4] = {x[i].vl.x, x[i].vl.y, x[i].vl.z, x[i].vl.w};
            if (valid < kBlock) {  // what lies behind the last token may be anything
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t keep = halves_below(8 * quarter + 2 * e, valid);
                    sc[e] &= keep;
                    lo[e] &= keep;
                }
            }
            const bool odd = ballot(is_odd(pair_max(pair_max(sc[0], sc[1]), pair_max(sc[2], sc[3])))) != 0;
            if (tree < kBlock) {
                uint32_t bits = 0;  // of the lane's eight tokens
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int t = 8 * quarter + 2 * e;
                    const bool b0 = t >= tree && (sc[e] & 0xFFFFu) >= 0x7C00u, b1 = t + 1 >= tree && sc[e] >= 0x7C000000u;
                    bits |= (uint32_t)b0 << (2 * e) | (uint32_t)b1 << (2 * e + 1);
                    const uint32_t keep = (b0 ? 0u : 0xFFFFu) | (b1 ? 0u : 0xFFFF0000u);
                    sc[e] &= keep;
                    lo[e] &= keep;
                }
                uint32_t all = 0;
#pragma unroll
                for (int q = 0; q < 4; ++q) all |= (uint32_t)__builtin_amdgcn_readlane((int)bits, 16 * q) << (8 * q);
                if (lane == 0) O.bad[task] = all;
            }
            const uint4 s4 = make_uint4(sc[0], sc[1], sc[2], sc[3]), l4 = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            half8_t v0 = values_of(M, x[i].v.x, s4, l4), v1 = values_of(M, x[i].v.y, s4, l4);
            if (odd) {
                const uint4 s2 = make_uint4(halves_of(sc[0]), halves_of(sc[1]), halves_of(sc[2]), halves_of(sc[3]));
                const uint4 l2 = make_uint4(halves_of(lo[0]), halves_of(lo[1]), halves_of(lo[2]), halves_of(lo[3]));
                v0 = values_of(M, x[i].v.x, s2, l2);
                v1 = values_of(M, x[i].v.y, s2, l2);
                if (lane == 0) O.odd[task] = O0->any_odd = blk0 + 1;
            }
            O.v[2 * task][lane] = __builtin_bit_cast(uint4, v0);
            O.v[2 * task + 1][lane] = __builtin_bit_cast(uint4, v1);
        }
    };
    uint32_t there = fetch(begin), there_next = 0;
    if (threadIdx.x < 2 * kStep) {
        Operands& O = L[threadIdx.x / kStep][threadIdx.x % kStep];
        O.any_odd = O.odd[0] = O.odd[1] = O.odd[2] = O.odd[3] = 0;
    }
    RowState<RT> R;
    R.start(A, rows, nodes, hk, r0, lane);
    __syncthreads();
    stage(L[0], begin, there);
    if (begin + kStep < end) there_next = fetch(begin + kStep);
    __syncthreads();
    int side = 0;
    for (int blk = begin; blk < end; blk += kStep) {
        const Operands* const O = L[side];
        side ^= 1;
        const int any_odd = O->any_odd;
        const uint32_t here = there;
        if (blk + kStep < end) stage(L[side], blk + kStep, there_next);
        there = there_next;
        if (blk + 2 * kStep < end) there_next = fetch(blk + 2 * kStep);
        if (here && active) {
            const bool odd = __builtin_amdgcn_readfirstlane(any_odd) == blk + 1;
#pragma unroll
            for (int b = 0; b < kStep; ++b) {
                if (!(here >> b & 1)) continue;
                const Operands& B = O[b];
                const int valid = valid_of(blk + b, true), tree = context - (blk + b) * kBlock;
                half8_t p[RT], v[8];
                uint32_t visible[RT];
                R.template weights<true>(
                    p, visible, valid, tree, quarter,
                    [&](int j, int g) __attribute__((always_inline)) { return __builtin_bit_cast(half8_t, B.k[j][g][lane]); },
                    [&](int g) __attribute__((always_inline)) { return reinterpret_cast<const uint4*>(B.scale)[4 * g + quarter]; },
                    [&](int j) __attribute__((always_inline)) { return B.low[quarter * kBlock + token_of(n, j)]; },
                    [&]() __attribute__((always_inline)) {  // on their way during the softmax
#pragma unroll
                        for (int ct = 0; ct < 8; ++ct) v[ct] = __builtin_bit_cast(half8_t, B.v[ct][lane]);
                    },
                    [&](int rt, int i) __attribute__((always_inline)) {  // the row tile's products between the next one's weights
                        R.add_one(2 * i, rt, v[2 * i], p);
                        R.add_one(2 * i + 1, rt, v[2 * i + 1], p);
                    });
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int ct = 0; ct < 8; ++ct) R.add_one(ct, RT - 1, v[ct], p);
                __builtin_amdgcn_s_setprio(0);
                if (tree < kBlock || odd) {  // (rare)
                    if (odd)  // the products again of values that are halves
#pragma unroll
                        for (int ct = 0; ct < 8; ++ct)
                            if (__builtin_amdgcn_readfirstlane(B.odd[ct >> 1]) == blk + 1) R.add(ct, __builtin_bit_cast(half8_t, B.v[ct][lane]), p);
                    if (tree < kBlock && (B.bad[0] | B.bad[1] | B.bad[2] | B.bad[3]) != 0)
                        R.add_bad(visible, [&](int g) __attribute__((always_inline)) { return B.bad[g]; });
                }
            }
        }
        __syncthreads();
    }
    if (active) R.finish(A, rows, hk, r0, wave * kWaveRows, kRows, record, lane);
}

// A workgroup's run of blocks, column by column: work(sequence, column, first and last block, record or -1).
template <class Work>
__device__ __forceinline__ void run_of(const TreeArgs& A, int rows_each, Work work) {
    const int all = sum_units(A, 0, rows_each).all, run = run_length(A, all);
    const int group = blockIdx.x, start = group * run;
    int left = min(run, all - start);
    if (left <= 0) return;
    const Item it = find_item(start, A.S, [&](int s) { return A.units(s, rows_each); });
    int s = it.seq;
    if (s < 0) return;
    int blocks = A.blocks(s), column = it.index / blocks, begin = it.index - column * blocks;
    int columns = A.chunks(s, rows_each) * A.pool.heads;
    for (bool first = true;; first = false) {
        const int count = min(left, blocks - begin);
        work(s, column, begin, begin + count, count == blocks ? -1 : 2 * group + !first);
        left -= count;
        if (left <= 0) return;
        begin = 0;
        if (++column == columns) {
            column = 0;
            do {
                if (++s == A.S) return;
                blocks = A.blocks(s);
                columns = A.chunks(s, rows_each) * A.pool.heads;
            } while (blocks == 0 || columns == 0);
        }
    }
}

template <int RT>
__global__ void __launch_bounds__(kWave, kWavesPerSimd) tree_alone_kernel(TreeArgs A) {
    __shared__ OneWave L;
    run_of(A, RT * kTileRows, [&](int s, int column, int begin, int end, int record) __attribute__((always_inline)) {
        work_alone<RT>(A, L, s, column, begin, end, record);
    });
}
template <int WAVES>
__global__ void __launch_bounds__(WAVES * kWave, kWavesPerSimd) tree_together_kernel(TreeArgs A) {
    __shared__ Operands L[2][kStep];
    run_of(A, WAVES * 2 * kTileRows, [&](int s, int column, int begin, int end, int record) __attribute__((always_inline)) {
        work_together<WAVES>(A, L, s, column, begin, end, record);
    });
}

// Joins the records of columns that several workgroups worked on, ROWS rows of a sequence and KV head per workgroup: 16
// threads a row, eight channels each, SPLIT such sets taking the records in turns, eight at a time.  Rows that nobody
// worked on get zeros; the workgroups behind the last item take the rows of no sequence.
template <int ROWS, int SPLIT>
__global__ void __launch_bounds__(ROWS * 16 * SPLIT) tree_merge_kernel(TreeArgs A) {
    constexpr int kSet = ROWS * 16, kAll = kSet * SPLIT;
    __shared__ float s_top[SPLIT][ROWS], s_total[SPLIT][ROWS];
    __shared__ float4 s_o[SPLIT > 1 ? SPLIT - 1 : 1][2][kSet];
    const int hk = (int)(blockIdx.x % A.pool.heads), item = (int)(blockIdx.x / A.pool.heads), tid = threadIdx.x;
    const Item it = find_item(item, A.S, [&](int s) { return (int)(((long)sequence_rows(A.offsets, s, A.N).count * A.G + ROWS - 1) / ROWS); });
    if (it.seq < 0) {
        if (!A.clear_rest) return;
        const int spares = (int)(gridDim.x / A.pool.heads) - (item - it.index);
        const int begin = min(max(A.offsets[0], 0), A.N), end = min(max(A.offsets[A.S], begin), A.N);
        const long pieces = (long)A.G * (kDim / 8), rest = (begin + A.N - end) * pieces;
        for (long i = (long)it.index * kAll + tid; i < rest; i += (long)spares * kAll) {
            const long r = i / pieces, row = r < begin ? r : end + r - begin;
            reinterpret_cast<uint4*>(A.out + (row * A.Hq + (long)hk * A.G) * kDim)[i - r * pieces] = make_uint4(0, 0, 0, 0);
        }
        return;
    }
    const int s = it.seq, set = tid / kSet, row = tid / 16 % ROWS, part = tid % 16;
    const Rows rows = sequence_rows(A.offsets, s, A.N);
    const int r = it.index * ROWS + row, node = r / A.G, blocks = A.blocks(s);
    const bool real = r < rows.count * A.G, worked = node < A.max_nodes;
    uint4* const out = reinterpret_cast<uint4*>(A.out + ((long)(rows.first + node) * A.Hq + hk * A.G + r - node * A.G) * kDim) + part;
    if (real && set == 0 && (blocks == 0 || !worked) && (worked || A.clear_rest)) *out = make_uint4(0, 0, 0, 0);
    if (blocks == 0 || it.index * ROWS >= A.max_nodes * A.G) return;
    const Sums sums = sum_units(A, s, A.rows_of_chunk);
    const int run = run_length(A, sums.all), in_chunk = r % A.rows_of_chunk;
    const int start = sums.before + (hk * A.chunks(s, A.rows_of_chunk) + it.index * ROWS / A.rows_of_chunk) * blocks;
    const int first = start / run, records = (start + blocks - 1) / run - first + 1;
    if (records <= 1) return;
    const bool late = first * run != start;  // the first workgroup's record is that of its last column
    float top = -__FLT_MAX__, total = 0.0f;
    float4 o0 = make_float4(0, 0, 0, 0), o1 = o0;
    for (int i0 = set; i0 < records; i0 += 8 * SPLIT) {
        float4 x[8][2];
        float2 ml[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int i = min(i0 + SPLIT * j, records - 1);
            const long rec = (long)(2 * (first + i) + (i == 0 && late)) * A.rows_of_chunk + in_chunk;
            const float4* const src = reinterpret_cast<const float4*>(A.part + rec * kDim) + 2 * part;
            x[j][0] = src[0];
            x[j][1] = src[1];
            ml[j] = A.stat[rec];
        }
        float most = top;
#pragma unroll
        for (int j = 0; j < 8; ++j) most = fmaxf(most, ml[j].x);
        const float alpha = __builtin_amdgcn_exp2f(top - most);
        o0.x *= alpha, o0.y *= alpha, o0.z *= alpha, o0.w *= alpha;
        o1.x *= alpha, o1.y *= alpha, o1.z *= alpha, o1.w *= alpha;
        total *= alpha;
        top = most;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (i0 + SPLIT * j >= records || ml[j].y == 0.0f) continue;  // saw nothing (a NaN goes on)
            const float a = __builtin_amdgcn_exp2f(ml[j].x - top);
            o0.x += a * x[j][0].x, o0.y += a * x[j][0].y, o0.z += a * x[j][0].z, o0.w += a * x[j][0].w;
            o1.x += a * x[j][1].x, o1.y += a * x[j][1].y, o1.z += a * x[j][1].z, o1.w += a * x[j][1].w;
            total += a * ml[j].y;
        }
    }
    if (SPLIT > 1) {
        if (part == 0) {
            s_top[set][row] = top;
            s_total[set][row] = total;
        }
        if (set > 0) {
            s_o[set - 1][0][tid % kSet] = o0;
            s_o[set - 1][1][tid % kSet] = o1;
        }
        __syncthreads();
        if (set > 0) return;
        float most = top;
#pragma unroll
        for (int i = 1; i < SPLIT; ++i) most = fmaxf(most, s_top[i][row]);
        const float alpha = __builtin_amdgcn_exp2f(top - most);
        o0.x *= alpha, o0.y *= alpha, o0.z *= alpha, o0.w *= alpha;
        o1.x *= alpha, o1.y *= alpha, o1.z *= alpha, o1.w *= alpha;
        total *= alpha;
#pragma unroll
        for (int i = 1; i < SPLIT; ++i) {
            if (s_total[i][row] == 0.0f) continue;
            const float a = __builtin_amdgcn_exp2f(s_top[i][row] - most);
            const float4 y0 = s_o[i - 1][0][tid], y1 = s_o[i - 1][1][tid];
            o0.x += a * y0.x, o0.y += a * y0.y, o0.z += a * y0.z, o0.w += a * y0.w;
            o1.x += a * y1.x, o1.y += a * y1.y, o1.z += a * y1.z, o1.w += a * y1.w;
            total += a * s_total[i][row];
        }
    }
    if (!real || !worked) return;
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    *out = make_uint4(pack_results(o0.x * inv, o0.y * inv), pack_results(o0.z * inv, o0.w * inv), pack_results(o1.x * inv, o1.y * inv),
                      pack_results(o1.z * inv, o1.w * inv));
}

// Rows of a workgroup: what the widest tree brings, 256 at most.
int chunk_rows(int G, int max_nodes) {
    const long rows = (long)G * max_nodes;
    return rows <= 16 ? 16 : rows <= 64 ? 32 : rows <= 128 ? 128 : 256;
}
int waves_of(int rows) { return rows <= 32 ? 1 : rows / 32; }

// Units when every sequence has the widest tree (offsets that fall may bring more than N rows in all).
long most_units(int S, int Hk, int G, long max_length, int max_nodes) {
    const long rows = chunk_rows(G, max_nodes), blocks = (max_length + kBlock - 1) / kBlock;
    return blocks * Hk * (((long)max_nodes * G + rows - 1) / rows) * S;
}
// Workgroups: as many as the chip holds at once, or one per unit when there are fewer.
long tree_groups(int S, long N, int Hk, int G, long max_length, int max_nodes) {
    const long rows = chunk_rows(G, max_nodes), blocks = (max_length + kBlock - 1) / kBlock;
    const long chunks = (N * G + rows - 1) / rows + S, widest = most_units(S, Hk, G, max_length, max_nodes);
    const long units = blocks * Hk * chunks < widest ? blocks * Hk * chunks : widest, most = kMostWaves / waves_of(rows);
    return units < 1 ? 1 : units < most ? units : most;
}

// Tiles of rows that S sequences of N rows in all can bring, and one that is always free.
long merge_items(long N, long G, int S, int rows) { return N * G / rows + S + 1; }

}  // namespace

extern "C" int64_t reskv_int4_tree_workspace_bytes(int S, int64_t N, int Hq, int Hk, int64_t max_length, int max_nodes) {
    if (S < 1 || N < 1 || N >= (1LL << 30) || Hk < 1 || Hq < 1 || Hq % Hk != 0 || max_length < 0 || max_length >= (1LL << 31) ||
        max_nodes < 1 || max_nodes > kNodes || Hq / Hk >= (1 << 20))
        return 0;
    const int G = Hq / Hk;
    return tree_groups(S, N, Hk, G, max_length, max_nodes) * 2 * chunk_rows(G, max_nodes) * (kDim + 2) * 4;
}

extern "C" int reskv_int4_tree_attention(const void* q, const void* pages, int64_t num_pages, int page_tokens,
                                         const int32_t* table, int table_width, const int32_t* lengths, const int32_t* offsets,
                                         const uint64_t* seen, int S, int64_t N, int Hq, int Hk, float scaling,
                                         int64_t max_length, int max_nodes, int clear_rest, void* out, void* workspace,
                                         int64_t workspace_bytes, void* stream) {
    RESKV_REQUIRE(q && lengths && offsets && out, "null pointer");
    if (!pool_ok(pages, num_pages, page_tokens, Hk, table, table_width)) return 1;
    RESKV_REQUIRE(S > 0 && N > 0 && N < (1LL << 30) && Hq > 0 && Hq % Hk == 0, "bad sizes (sequences %d, rows %ld, query heads %d, KV heads %d)",
                  S, (long)N, Hq, Hk);
    RESKV_REQUIRE(max_nodes >= 1 && max_nodes <= kNodes, "a tree has 1 to %d nodes", kNodes);
    RESKV_REQUIRE(max_length >= 0, "max_length must not be negative");
    RESKV_REQUIRE(scaling > 0.0f && scaling < 1e30f, "scaling must be positive and below 1e30");
    RESKV_REQUIRE(aligned16(q) && aligned16(out) && aligned16(workspace), "tensors must be 16-byte aligned");
    const long most = (long)table_width * page_tokens;
    if (max_length > most) max_length = most;
    const int G = Hq / Hk;
    // units and rows are counted in 32 bits; the last wave's run may end behind the last unit
    RESKV_REQUIRE(most_units(S, Hk, G, max_length, max_nodes) < (1L << 30) && G < (1 << 20),
                  "too many tokens: blocks of %d x KV heads x chunks of rows must stay below 2^30", kBlock);
    // The fewer the rows, the more threads of the merge take each one's records, which come from the whole chip then: 8 nodes of 32 heads
    // after 20000 tokens (256 records a row) 32 us for both kernels with 16 sets and 46 with four, five trees of 1 to 61 nodes 129 with
    // four and 139 with 16.
    const long rows_all = (long)N * Hq;
    const auto merge = rows_all <= 1024 ? tree_merge_kernel<4, 16> : rows_all <= 8192 ? tree_merge_kernel<16, 4> : tree_merge_kernel<16, 1>;
    const int merge_threads = rows_all <= 8192 ? 1024 : 256;
    const long merge_groups = merge_items(N, G, S, rows_all <= 1024 ? 4 : 16) * Hk;
    RESKV_REQUIRE(merge_groups < kLaunchThreads / merge_threads, "too many tokens: %ld nodes of %d sequences for %d KV heads pass a launch's 2^32 threads",
                  (long)N, S, Hk);
    RESKV_REQUIRE(workspace && workspace_bytes >= reskv_int4_tree_workspace_bytes(S, N, Hq, Hk, max_length, max_nodes), "the workspace is too small");
    const int rows = chunk_rows(G, max_nodes);
    TreeArgs A{};
    A.pool = make_pool(pages, num_pages, page_tokens, Hk, table, table_width);
    A.q = (const uint16_t*)q;
    A.lengths = lengths;
    A.offsets = offsets;
    A.seen = seen;
    A.out = (uint16_t*)out;
    A.S = S;
    A.N = (int)N;
    A.Hq = Hq;
    A.G = G;
    A.groups = (int)tree_groups(S, N, Hk, G, max_length, max_nodes);
    A.part = (float*)workspace;
    A.stat = (float2*)(A.part + (long)A.groups * 2 * rows * kDim);
    A.max_length = (int)max_length;
    A.max_nodes = max_nodes;
    A.rows_of_chunk = rows;
    A.clear_rest = clear_rest;
    A.c = scaling * 1.4426950408889634f;
    const auto kernel = rows == 16 ? tree_alone_kernel<1> : rows == 32 ? tree_alone_kernel<2> : rows == 128 ? tree_together_kernel<4> : tree_together_kernel<8>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)A.groups), dim3(kWave * waves_of(rows)), 0, (hipStream_t)stream, A);
    if (reskv_host::check_launch("tree_kernel")) return 1;
    hipLaunchKernelGGL(merge, dim3((unsigned)merge_groups), dim3((unsigned)merge_threads), 0, (hipStream_t)stream, A);
    return reskv_host::check_launch("tree_merge_kernel");
}
