// Attention of the nodes of drafted trees over a paged cache of 4-bit keys and values (include/reskv_drafts.h).
//
// Row r of a sequence and KV head is node r / G of query head r % G of the head's group; a tile has 16 rows, a wave RT
// tiles.  For 32 tokens and each of the four groups g of 32 channels, on v_mfma_f32_16x16x32_f16,
//   S_g^T [token][row] = K_g Q_g^T, codes as fp16 by masking alone (see int4.hip), and
//   S^T = low q-sum^T + sum_g scale[token, g] S_g^T,
// the first term on v_mfma_f32_16x16x4_f32 (its inner dimension is the four groups), the others as one mixed fp32 / fp16
// multiply-add per score and group, so that keys are not rounded.  The rows of the K operand are taken in an order of
// tokens that leaves lane (quarter q, row n) with the scores of the tokens 8 q .. 8 q + 7: the order in which
// V's codes lie in a lane.  Softmax and its statistics are then a lane's own but for the maximum, and the weights are the B
// operand of
//   O^T [channel][row] += V^T P^T
// as they are, without the LDS.  V = code * scale + low is rounded to fp16 once (the row that reskv_int4_gather gives): the
// work of that is shared by the rows of a wave.
//
// Scores, softmax and sums are fp32.  Weights are 2^9 exp2(x - m), m at most 6 below the row's largest score so far, rounded
// to fp16 for the product and summed as rounded: eleven bits down to 2^-23 of the largest weight.
#include "int4.h"
#include "reskv_drafts.h"

using namespace reskv;

namespace {

constexpr int kNodes = RESKV_DRAFT_NODES;
constexpr int kWavesPerSimd = 2;
constexpr int kMostWaves = 1024 * kWavesPerSimd;  // 256 CUs of 4 SIMDs
constexpr float kWeightBits = 9.0f, kSlack = 6.0f;
constexpr int kTileRows = 16;

// Work: a column is (sequence, KV head, chunk of rows), as many blocks of 32 tokens long as the sequence; the columns
// lie one behind the other and every wave takes an equal run of blocks.  A column that lies in one run is written
// out at once; of the others every wave leaves a record, of its first column at 2 wave, of its last at 2 wave + 1.
struct TreeArgs {
    Pool pool;
    const uint16_t* q;       // [N, Hq, 128]
    const int32_t *lengths, *offsets;
    const uint64_t* seen;    // [N] or null
    uint16_t* out;           // [N, Hq, 128]
    float* part;             // [2 waves, rows, 128]: weighted values
    float2* stat;            // [2 waves, rows]: reference of the weights, their sum
    int S, N, Hq, G, waves, max_length, max_nodes, clear_rest;
    float c;                 // scaling * log2(e)

    __device__ __forceinline__ int tokens(int s) const { return min(max(lengths[s], 0), max_length); }
    __device__ __forceinline__ int blocks(int s) const { return (tokens(s) + kBlock - 1) / kBlock; }
    __device__ __forceinline__ Rows rows(int s) const {
        const Rows r = sequence_rows(offsets, s, N);
        return {r.first, min(r.count, max_nodes)};
    }
    template <int ROWS>
    __device__ __forceinline__ int chunks(int s) const { return (rows(s).count * G + ROWS - 1) / ROWS; }
    template <int ROWS>
    __device__ __forceinline__ int units(int s) const { return blocks(s) * chunks<ROWS>(s) * pool.heads; }
};

// Units (blocks of columns) of the sequences before s, and of all.
struct Sums {
    int before, all;
};
template <int ROWS>
__device__ __forceinline__ Sums sum_units(const TreeArgs& A, int s) {
    int before = 0, all = 0;
    for (int i = lane_id(); i < A.S; i += kWave) {
        const int n = A.units<ROWS>(i);
        all += n;
        before += i < s ? n : 0;
    }
    return {wave_sum_int(before), wave_sum_int(all)};
}
__device__ __forceinline__ int run_length(const TreeArgs& A, int all) { return max((all + A.waves - 1) / A.waves, 1); }

// One block as a lane takes it.
struct TreeBlock {
    uint4 k[2];      // tokens token_of(j), channels 8 quarter + [0, 8) of the four groups
    uint32_t ks[2];  // their scale and low of group `quarter`
    uint4 v[2];      // channels 16 (4 i + j) + lane % 16 (dword j), tokens 8 quarter + [0, 8)
    uint32_t vs, vl; // scales and lowest values of group lane / 16, tokens 2 (lane % 16) + [0, 2)
};
// Token of a lane's row in tile j of K: rows 4 q .. 4 q + 3 are the tokens 8 q + 4 j .. + 3.
__device__ __forceinline__ int token_of(int n, int j) { return 8 * (n >> 2) + 4 * j + (n & 3); }

__device__ __forceinline__ void load_block(TreeBlock& b, const char* p, int lane) {
    const int n = lane & 15, quarter = lane >> 4;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int t = token_of(n, j);
        b.k[j] = reinterpret_cast<const uint4*>(p)[(t >> 4) * 64 + quarter * 16 + (t & 15)];
        b.ks[j] = reinterpret_cast<const uint32_t*>(p + kKScale)[((t >> 4) * 4 + quarter) * 16 + (t & 15)];
    }
    b.v[0] = reinterpret_cast<const uint4*>(p + kVCodes)[lane];
    b.v[1] = reinterpret_cast<const uint4*>(p + kVCodes)[64 + lane];
    b.vs = reinterpret_cast<const uint32_t*>(p + kVScale)[lane];
    b.vl = reinterpret_cast<const uint32_t*>(p + kVLow)[lane];
}

// Eight values code * scale + low in fp16 of a dword of codes, `s` and `l` being the scales and lowest values of its
// elements: the codes become 1024 + code, or 1024 + 16 code, by masking, and code exactly from that.
__device__ __forceinline__ half8_t values_of(uint32_t d, const uint4& s, const uint4& l) {
    const half2_t sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f}, back = {(_Float16)-64.0f, (_Float16)-64.0f};
    const half2_t base = {(_Float16)1024.0f, (_Float16)1024.0f};
    const uint32_t e = d >> 8, m = 0x64006400u;
    const half2_t c0 = __builtin_bit_cast(half2_t, (d & 0x000F000Fu) | m) - base, c2 = __builtin_bit_cast(half2_t, (e & 0x000F000Fu) | m) - base;
    const half2_t c1 = __builtin_elementwise_fma(__builtin_bit_cast(half2_t, (d & 0x00F000F0u) | m), sixteenth, back);
    const half2_t c3 = __builtin_elementwise_fma(__builtin_bit_cast(half2_t, (e & 0x00F000F0u) | m), sixteenth, back);
    auto h = [](uint32_t w) __attribute__((always_inline)) { return __builtin_bit_cast(half2_t, w); };
    const half2_t r0 = __builtin_elementwise_fma(c0, h(s.x), h(l.x)), r1 = __builtin_elementwise_fma(c1, h(s.y), h(l.y));
    const half2_t r2 = __builtin_elementwise_fma(c2, h(s.z), h(l.z)), r3 = __builtin_elementwise_fma(c3, h(s.w), h(l.w));
    return half8_t{r0[0], r0[1], r1[0], r1[1], r2[0], r2[1], r3[0], r3[1]};
}

// A value past fp16's largest, which code * scale + low can reach by the rounding of the scale, is that largest (a NaN
// goes on).
__device__ __forceinline__ half8_t within_fp16(half8_t v) {
    const _Float16 top = (_Float16)65504.0f;
    const half8_t most = {top, top, top, top, top, top, top, top};
    return __builtin_elementwise_maximum(__builtin_elementwise_minimum(v, most), -most);
}

template <int RT>
__device__ __forceinline__ void work_on_column(const TreeArgs& A, uint32_t* s_ks, uint32_t* s_vs, int s, int column, int begin,
                                               int end, int record) {
    constexpr int kRows = RT * kTileRows;
    const int lane = threadIdx.x, n = lane & 15, quarter = lane >> 4;
    const Rows rows = A.rows(s);
    const int chunks = A.chunks<kRows>(s), hk = column / chunks, r0 = (column - hk * chunks) * kRows;
    const int total_rows = rows.count * A.G, length = A.tokens(s), context = length - rows.count;

    int entry0 = begin / A.pool.blocks, entry = 0, inside = begin - entry0 * A.pool.blocks, numbers = 0;
    auto fetch_numbers = [&]() { numbers = A.pool.table[(long)s * A.pool.width + min(entry0 + lane, A.pool.width - 1)]; };
    auto fetch = [&](TreeBlock& x) {
        const char* p = A.pool.in_page(__builtin_amdgcn_readlane(numbers, entry), inside, hk);
        load_block(x, p ? p : A.pool.pages, lane);
        if (++inside == A.pool.blocks) {
            inside = 0;
            if (++entry == kWave) {
                entry0 += kWave;
                entry = 0;
                fetch_numbers();
            }
        }
        return p != nullptr;
    };
    TreeBlock x0, x1;
    fetch_numbers();
    bool there0 = fetch(x0);

    // Q: lane (row n, quarter): channels 32 g + 8 quarter + [0, 8) of each group, brought to the row's own power of two so
    // that the sixteenth of an element, which meets codes times 2^-20, keeps its bits
    half8_t qf[RT][4];
    float qs[RT], back[RT];  // sum of group `quarter`'s channels; what brings the row's scores back
    uint64_t sees[RT];       // the row's nodes
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = r0 + rt * kTileRows + n, node = r / A.G;
        const bool real = r < total_rows;
        const long row = (long)(rows.first + node) * A.Hq + hk * A.G + r - node * A.G;
        float top = 0.0f, sum[4];
        uint4 raw[4] = {};
        if (real) {
#pragma unroll
            for (int g = 0; g < 4; ++g) raw[g] = reinterpret_cast<const uint4*>(A.q + row * kDim)[4 * g + quarter];
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const uint32_t w[4] = {raw[g].x, raw[g].y, raw[g].z, raw[g].w};
            sum[g] = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = h2f((uint16_t)(w[e >> 1] >> (16 * (e & 1))));
                top = fmaxf(top, fabsf(x));
                sum[g] += x;
            }
        }
        top = swap_max(top);
        const float up = top > 0.0f && top < INFINITY ? ldexpf(1.0f, 14 - ilogbf(top)) : 1.0f;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const uint32_t w[4] = {raw[g].x, raw[g].y, raw[g].z, raw[g].w};
#pragma unroll
            for (int e = 0; e < 8; ++e)
                qf[rt][g][e] = (_Float16)(h2f((uint16_t)(w[e >> 1] >> (16 * (e & 1)))) * (e & 2 ? up * 0.0625f : up));
            sum[g] = swap_sum16(sum[g], sum[g]);
            sum[g] = swap_sum32(sum[g], sum[g]);
        }
        qs[rt] = (quarter == 0 ? sum[0] : quarter == 1 ? sum[1] : quarter == 2 ? sum[2] : sum[3]) * (up * 0x1p-24f);
        back[rt] = A.c * (0x1p24f / up);
        const uint64_t all = rows.count < 64 ? (1ull << rows.count) - 1 : ~0ull;
        sees[rt] = !real ? 0 : (A.seen ? A.seen[rows.first + node] : (2ull << node) - 1) & all;
    }

    float4_t acc[RT][8];  // channels 16 ct + 4 quarter + i of row n
    float m[RT], l[RT];   // reference of the row's weights, this lane's share of their sum
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -__FLT_MAX__;
        l[rt] = 0.0f;
#pragma unroll
        for (int ct = 0; ct < 8; ++ct) acc[rt][ct] = {0.0f, 0.0f, 0.0f, 0.0f};
    }

    auto work = [&](TreeBlock& x, int blk, bool there) __attribute__((always_inline)) {
        if (!there) return;  // its tokens are not there
        const int valid = min(kBlock, length - blk * kBlock), tree = context - blk * kBlock;  // tokens; where the nodes begin
        const bool edge = tree < kBlock;  // some tokens are nodes, or none
        if (valid < kBlock) {  // what lies behind the last token may be anything
            const int t = 2 * n;
            const uint32_t keep = (t < valid ? 0xFFFFu : 0u) | (t + 1 < valid ? 0xFFFF0000u : 0u);
            x.vs &= keep;
            x.vl &= keep;
        }
        // Scales of 2^12 and more, NaN and infinity among them: values may pass fp16's largest
        const bool odd = ballot((x.vs & 0xFFFFu) >= 0x6C00u || x.vs >= 0x6C000000u) != 0;
        uint64_t bad0 = 0, bad1 = 0;  // nodes (even and odd tokens, 16 a group) whose values are no numbers
        if (odd && edge) {
            const int t = 2 * n;
            const bool b0 = t >= tree && (x.vs & 0xFFFFu) >= 0x7C00u, b1 = t + 1 >= tree && x.vs >= 0x7C000000u;
            bad0 = ballot(b0);
            bad1 = ballot(b1);
            const uint32_t keep = (b0 ? 0u : 0xFFFFu) | (b1 ? 0u : 0xFFFF0000u);
            x.vs &= keep;  // zeros to the rows that do not see them, added apart to the others
            x.vl &= keep;
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) s_ks[quarter * kBlock + token_of(n, j)] = x.ks[j];
        s_vs[lane] = x.vs;
        s_vs[64 + lane] = x.vl;
        wave_sync();

        float4_t score[RT][2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float low = h2f((uint16_t)(x.ks[j] >> 16));
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
                score[rt][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(low, qs[rt], float4_t{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
        }
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t kd = g == 0 ? x.k[j].x : g == 1 ? x.k[j].y : g == 2 ? x.k[j].z : x.k[j].w;
                const half8_t kf = operand(kd);
                const uint4 sc = *reinterpret_cast<const uint4*>(&s_ks[g * kBlock + 8 * quarter + 4 * j]);
                const uint32_t w[4] = {sc.x, sc.y, sc.z, sc.w};
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    const float4_t d = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[rt][g], float4_t{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; ++i) score[rt][j][i] = __builtin_fmaf(d[i], h2f((uint16_t)w[i]), score[rt][j][i]);
                }
            }

        uint32_t sees_block[RT];
        if (edge || valid < kBlock) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                uint32_t bits = tree <= 0 ? (tree > -64 ? (uint32_t)(sees[rt] >> -tree) : 0u)
                                          : tree < kBlock ? (uint32_t)(sees[rt] << tree) | ((1u << tree) - 1u) : ~0u;
                if (valid < kBlock) bits &= (1u << valid) - 1u;
                sees_block[rt] = bits;
                const uint32_t mine = bits >> (8 * quarter);
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (!((mine >> (4 * j + i)) & 1u)) score[rt][j][i] = -INFINITY;
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
        half8_t p[RT];
        const half2_t ones = {(_Float16)1.0f, (_Float16)1.0f};
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const float shift = kWeightBits - m[rt];
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const half2_t w = {(_Float16)__builtin_amdgcn_exp2f(__builtin_fmaf(score[rt][e >> 2][e & 3], back[rt], shift)),
                                   (_Float16)__builtin_amdgcn_exp2f(__builtin_fmaf(score[rt][e >> 2][(e & 3) + 1], back[rt], shift))};
                sum = __builtin_amdgcn_fdot2(w, ones, sum, false);
                p[rt][e] = w[0];
                p[rt][e + 1] = w[1];
            }
            l[rt] += sum;
        }
#pragma unroll
        for (int ct = 0; ct < 8; ++ct) {
            const uint4 sc = *reinterpret_cast<const uint4*>(&s_vs[(ct >> 1) * 16 + 4 * quarter]);
            const uint4 lo = *reinterpret_cast<const uint4*>(&s_vs[64 + (ct >> 1) * 16 + 4 * quarter]);
            const uint4& codes = x.v[ct >> 2];
            const int at = ct & 3;
            half8_t v = values_of(at == 0 ? codes.x : at == 1 ? codes.y : at == 2 ? codes.z : codes.w, sc, lo);
            if (odd) v = within_fp16(v);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) acc[rt][ct] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p[rt], acc[rt][ct], 0, 0, 0);
        }
        if ((bad0 | bad1) != 0) {  // rare: the rows that see such a node get its NaN, in the channels of its group
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
                for (int t = 0; t < kBlock; ++t)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        if (((t & 1 ? bad1 : bad0) >> (16 * g + (t >> 1))) & 1u && (sees_block[rt] >> t) & 1u)
#pragma unroll
                            for (int i = 0; i < 4; ++i) acc[rt][2 * g][i] = acc[rt][2 * g + 1][i] = __builtin_nanf("");
        }
        wave_sync();
    };
    bool there1 = false;
    for (int blk = begin; blk < end; blk += 2) {
        if (blk + 1 < end) there1 = fetch(x1);
        work(x0, blk, there0);
        if (blk + 1 >= end) break;
        if (blk + 2 < end) there0 = fetch(x0);
        work(x1, blk + 1, there1);
    }

#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        float total = swap_sum16(l[rt], l[rt]);
        total = swap_sum32(total, total);
        const int at = rt * kTileRows + n, r = r0 + at, node = r / A.G;
        if (r >= total_rows) continue;
        if (record >= 0) {
            const long rec = (long)record * kRows + at;
            if (quarter == 0) A.stat[rec] = make_float2(m[rt], total);
            float4_t* const dst = reinterpret_cast<float4_t*>(A.part + rec * kDim) + quarter;
#pragma unroll
            for (int ct = 0; ct < 8; ++ct) dst[4 * ct] = acc[rt][ct];
        } else {
            const float inv = total == 0.0f ? 0.0f : 1.0f / total;
            uint2* const dst = reinterpret_cast<uint2*>(A.out + ((long)(rows.first + node) * A.Hq + hk * A.G + r - node * A.G) * kDim) + quarter;
#pragma unroll
            for (int ct = 0; ct < 8; ++ct)
                dst[4 * ct] = make_uint2(pack_halves(acc[rt][ct][0] * inv, acc[rt][ct][1] * inv), pack_halves(acc[rt][ct][2] * inv, acc[rt][ct][3] * inv));
        }
    }
    wave_sync();
}

template <int RT>
__global__ void __launch_bounds__(kWave, kWavesPerSimd) tree_kernel(TreeArgs A) {
    constexpr int kRows = RT * kTileRows;
    __shared__ __align__(16) uint32_t s_ks[4 * kBlock], s_vs[128];
    const int all = sum_units<kRows>(A, 0).all, run = run_length(A, all);
    const int wave = blockIdx.x, start = wave * run;
    int left = min(run, all - start);
    if (left <= 0) return;
    const Item it = find_item(start, A.S, [&](int s) { return A.units<kRows>(s); });
    int s = it.seq;
    if (s < 0) return;
    int blocks = A.blocks(s), column = it.index / blocks, begin = it.index - column * blocks;
    int columns = A.chunks<kRows>(s) * A.pool.heads;
    for (bool first = true;; first = false) {
        const int count = min(left, blocks - begin);
        work_on_column<RT>(A, s_ks, s_vs, s, column, begin, begin + count, count == blocks ? -1 : 2 * wave + !first);
        left -= count;
        if (left <= 0) return;
        begin = 0;
        if (++column == columns) {
            column = 0;
            do {
                if (++s == A.S) return;
                blocks = A.blocks(s);
                columns = A.chunks<kRows>(s) * A.pool.heads;
            } while (blocks == 0 || columns == 0);
        }
    }
}

// Joins the records of columns that several waves worked on, two (node, query head) rows per wave and four channels per lane;
// zeros for nodes that nobody worked on.
constexpr int kMergeRows = 2 * (kThreads / kWave);
template <int RT>
__global__ void __launch_bounds__(kThreads) tree_merge_kernel(TreeArgs A) {
    constexpr int kRows = RT * kTileRows;
    const int lane = threadIdx.x & 63, half = lane >> 5;
    const long row0 = ((long)blockIdx.x * (kThreads / kWave) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * 2;
    int first = 0, records = 0, r = 0;   // of the lane's row: its column's first wave, the waves, the row in its chunk
    bool late = false, zero = false;     // the first wave's record is its last one; the row gets zeros
    const long mine = row0 + half;
    const bool there = mine < (long)A.N * A.Hq;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const long row = row0 + h;
        if (row >= (long)A.N * A.Hq) break;
        const int at = (int)(row / A.Hq), head = (int)(row - (long)at * A.Hq);
        // the sequence of row `at`
        int s = -1, node = 0;
        for (int s0 = 0; s0 < A.S && s < 0; s0 += kWave) {
            const int i = s0 + lane;
            const Rows q = i < A.S ? sequence_rows(A.offsets, i, A.N) : Rows{0, 0};
            const uint64_t who = ballot(at >= q.first && at < q.first + q.count);
            if (who == 0) continue;
            const int of = __builtin_ctzll(who);
            s = s0 + of;
            node = at - __builtin_amdgcn_readlane(q.first, of);
        }
        if (s < 0 || node >= A.max_nodes) {
            if (half == h) zero = A.clear_rest;
            continue;
        }
        const int blocks = A.blocks(s);
        if (blocks == 0) {
            if (half == h) zero = true;
            continue;
        }
        const Sums sums = sum_units<kRows>(A, s);
        const int run = run_length(A, sums.all), hk = head / A.G, in = node * A.G + head - hk * A.G;
        const int start = sums.before + (hk * A.chunks<kRows>(s) + in / kRows) * blocks;
        if (half == h) {
            first = start / run;
            records = (start + blocks - 1) / run - first + 1;
            late = first * run != start;
            r = in % kRows;
        }
    }
    if (!there) return;
    uint2* const out = reinterpret_cast<uint2*>(A.out + mine * kDim) + (lane & 31);
    if (zero) *out = make_uint2(0, 0);
    if (records <= 1) return;
    auto record = [&](int i) { return (long)(2 * (first + i) + (i == 0 && late)) * kRows + r; };
    float top = -__FLT_MAX__, total = 0.0f, o[4] = {};
    for (int i0 = 0; i0 < records; i0 += 8) {
        float4 x[8];
        float2 ml[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const long rec = record(min(i0 + j, records - 1));
            x[j] = reinterpret_cast<const float4*>(A.part + rec * kDim)[lane & 31];
            ml[j] = A.stat[rec];
        }
        float most = top;
#pragma unroll
        for (int j = 0; j < 8; ++j) most = fmaxf(most, ml[j].x);
        const float alpha = __builtin_amdgcn_exp2f(top - most);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] *= alpha;
        total *= alpha;
        top = most;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (i0 + j >= records || ml[j].y == 0.0f) continue;  // saw nothing (a NaN goes on)
            const float a = __builtin_amdgcn_exp2f(ml[j].x - top);
            o[0] += a * x[j].x;
            o[1] += a * x[j].y;
            o[2] += a * x[j].z;
            o[3] += a * x[j].w;
            total += a * ml[j].y;
        }
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    *out = make_uint2(pack_halves(o[0] * inv, o[1] * inv), pack_halves(o[2] * inv, o[3] * inv));
}

// Tiles of rows of a wave: what the widest tree brings, two at most.
int tiles_of(int G, int max_nodes) { return G * max_nodes <= kTileRows ? 1 : 2; }

// Units when every sequence has the widest tree (offsets that fall may bring more than N rows in all).
long most_units(int S, int Hk, int G, long max_length, int max_nodes) {
    const long rows = tiles_of(G, max_nodes) * kTileRows, blocks = (max_length + kBlock - 1) / kBlock;
    return blocks * Hk * (((long)max_nodes * G + rows - 1) / rows) * S;
}
long tree_waves(int S, long N, int Hk, int G, long max_length, int max_nodes) {
    const long rows = tiles_of(G, max_nodes) * kTileRows, blocks = (max_length + kBlock - 1) / kBlock;
    const long chunks = (N * G + rows - 1) / rows + S, widest = most_units(S, Hk, G, max_length, max_nodes);
    const long units = blocks * Hk * chunks < widest ? blocks * Hk * chunks : widest;
    return units < 1 ? 1 : units < kMostWaves ? units : kMostWaves;
}

}  // namespace

extern "C" int64_t reskv_int4_tree_workspace_bytes(int S, int64_t N, int Hq, int Hk, int64_t max_length, int max_nodes) {
    if (S < 1 || N < 1 || N >= (1LL << 30) || Hk < 1 || Hq < 1 || Hq % Hk != 0 || max_length < 0 || max_length >= (1LL << 31) ||
        max_nodes < 1 || max_nodes > kNodes || Hq / Hk >= (1 << 20))
        return 0;
    const int G = Hq / Hk;
    return tree_waves(S, N, Hk, G, max_length, max_nodes) * 2 * tiles_of(G, max_nodes) * kTileRows * (kDim + 2) * 4;
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
    RESKV_REQUIRE(most_units(S, Hk, G, max_length, max_nodes) < (1L << 30) && G < (1 << 20) && N * Hq < kLaunchThreads / kWave,
                  "too many tokens: blocks of %d x KV heads x chunks of rows must stay below 2^30", kBlock);
    RESKV_REQUIRE(workspace && workspace_bytes >= reskv_int4_tree_workspace_bytes(S, N, Hq, Hk, max_length, max_nodes), "the workspace is too small");
    const int tiles = tiles_of(G, max_nodes);
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
    A.waves = (int)tree_waves(S, N, Hk, G, max_length, max_nodes);
    A.part = (float*)workspace;
    A.stat = (float2*)(A.part + (long)A.waves * 2 * tiles * kTileRows * kDim);
    A.max_length = (int)max_length;
    A.max_nodes = max_nodes;
    A.clear_rest = clear_rest;
    A.c = scaling * 1.4426950408889634f;
    hipLaunchKernelGGL(tiles == 1 ? tree_kernel<1> : tree_kernel<2>, dim3((unsigned)A.waves), dim3(kWave), 0, (hipStream_t)stream, A);
    if (reskv_host::check_launch("tree_kernel")) return 1;
    const long rows = (long)N * Hq;
    hipLaunchKernelGGL(tiles == 1 ? tree_merge_kernel<1> : tree_merge_kernel<2>, dim3((unsigned)((rows + kMergeRows - 1) / kMergeRows)),
                       dim3(kThreads), 0, (hipStream_t)stream, A);
    return reskv_host::check_launch("tree_merge_kernel");
}
