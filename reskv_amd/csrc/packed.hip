// Causal attention of packed sequences of different lengths (include/reskv_serving.h).
//
// One workgroup of eight waves per 256 rows of one KV head and sequence, where row r is
// query r / G of query head r % G of the head's group: short sequences and single tokens then fill
// the matrix cores' columns with the heads of a group, whatever G is.  A wave owns 32
// rows; keys are taken 64 at a time from double-buffered LDS.
//   S^T = K Q^T on v_mfma_f32_32x32x16_f16: lane (col = lane % 32, half = lane / 32)
//     holds its row's scores of keys 8 (i / 4) + 4 half + i % 4, i = 0..15, of a
//     32-key block, so the softmax needs one lane swap, and the fp16 weights are the
//     B operand of
//   O^T = V^T P^T as they are: its 16-key steps take the keys in the order in which
//     a lane holds them.
// The 16-byte pieces of a row of K are staged permuted, so that the rows' reads fall on different banks; V is
// staged transposed, in the order of keys of the weights, so that its operand is one 16-byte read
// (transposing reads run at half the rate).
//
// The two halves of a workgroup, a wave of each on every SIMD, are half a tile apart: one multiplies with K while
// the other does its softmax and multiplies with V, so that the vector ALU (about 830 cycles a tile and wave, half of
// them exponentials) works beside the matrix cores (1024).  One workgroup of 256 rows also fetches and stages K and V
// half as often as two of 128: 16384 tokens, 32 / 8 heads, 2.13 to 2.19 ms (1005 to 1030 TFLOP/s, by the card) against
// 2.41 with four waves that take no turns; 24 prompts of 16 to 1500 tokens 117 to 122 us, where four waves took 120.
//
// Bound: long prompts by the power that the matrix cores may draw: with zeros in K and V the same
// instructions take 1.75 ms, as a library product of 16384 x 16384 matrices makes 1761 TFLOP/s of zeros and 1277 of
// random numbers.  Short ones also by what a workgroup does alone on its CU at its start and end (about 6 us: its place
// among the offsets, the first tiles, its rows' way out).
//
// Scores, softmax and sums are fp32.  The weights are rounded to fp16 for the second product, and summed
// as rounded; they are 2^9 exp2(x - m) with m at most 6 (kSlack, in powers of two) below the row's largest score so far, so
// that a weight has fewer than fp16's eleven bits only when it is below 2^-23 of the largest, and is lost only below 2^-33.
// In two fp16 operands each, a rounded part and the rest, the weights keep 22 bits; outputs then differ from the ones of 32-bit
// weights by 2e-5 to 3e-5 instead of 1.5e-4 to 2e-4 (their own rounding to fp16 is 2.07e-4), and a long prompt takes 3.05 ms
// instead of 2.15, 24 prompts 151 us instead of 122, 3 chunks after 20000 tokens 169 instead of 126.
#include "serving.h"
#include "reskv_serving.h"

using namespace reskv;

namespace {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float16_t __attribute__((ext_vector_type(16)));

constexpr int kWaves = 8;
constexpr int kThreads = kWaves * kWave;
constexpr int kWaveRows = 32;
constexpr int kRows = kWaves * kWaveRows;
constexpr int kKeys = 64;           // keys per tile
constexpr int kVPitch = kKeys + 8;  // halves per staged row of V transposed: rows start on different banks
constexpr int kOutPitch = kDim + 8;
constexpr float kWeightBits = 9.0f;
constexpr float kSlack = 6.0f;      // how far a score may pass m before m moves up: weights stay within 2^15
constexpr int kRecord = kDim + 2;

struct PackedArgs {
    const uint16_t *q, *k, *v;
    uint16_t* out;               // [Nq, Hq, 128]
    const int32_t *q_offsets, *k_offsets;
    float* part;                 // split keys: [workgroups, record_rows, 128]: weighted values
    float2* stat;                // [workgroups, record_rows]: reference of the weights, their sum
    int32_t* length;             // tiles of keys of a part
    long q_token, q_head, k_token, k_head, v_token, v_head;  // strides in halves
    int sequences, Nq, Nk, Hq, Hk, G;
    int items, clear_rest;
    int groups;                  // split keys: workgroups of a KV head
    int record_rows;             // rows that a workgroup can have
    float c;                     // scaling * log2(e)
};

__device__ __forceinline__ uint32_t finite_or_zero(uint32_t pair) {
    return pair & (((pair & 0x7C00u) == 0x7C00u ? 0u : 0xFFFFu) | ((pair & 0x7C000000u) == 0x7C000000u ? 0u : 0xFFFF0000u));
}

// Item `index` of sequence `seq` (see find_item), and the sequence's rows.
struct Place {
    Item item;
    Rows q, k;
};

__device__ __forceinline__ int row_tiles(const PackedArgs& A, int queries) {
    return (int)(((long)queries * A.G + kRows - 1) / kRows);
}

__device__ __forceinline__ Place place_in_order(const PackedArgs& A, int t) {
    const Item it = find_item(t, A.sequences, [&](int s) { return row_tiles(A, sequence_rows(A.q_offsets, s, A.Nq).count); });
    if (it.seq < 0) return {it, {0, 0}, {0, 0}};
    return {it, sequence_rows(A.q_offsets, it.seq, A.Nq), sequence_rows(A.k_offsets, it.seq, A.Nk)};
}

// Item t in the order of their cost, the dearest first, so that the last ones to start are short: a tile's
// cost is its number among the sequence's, on top of what the keys in front of the queries cost.  One lane
// has each sequence; the cost of item t is found by halving, with one sum over the wave per step.
__device__ __forceinline__ Place place_by_cost(const PackedArgs& A, int t, const Rows& q, const Rows& k) {
    const int tiles = row_tiles(A, q.count), base = (int)((long)max(k.count - q.count, 0) * A.G / kRows);
    auto dearer = [&](int cost) __attribute__((always_inline)) {  // items of this lane's sequence that cost more: base + 1 .. base + tiles
        return min(max(base + tiles - cost, 0), tiles);
    };
    const int all = wave_sum_int(tiles);
    if (t >= all) return {{-1, t - all}, {0, 0}, {0, 0}};
    int low = 0, high = wave_max_int(base + tiles);  // items dearer than low: more than t; than high: at most t
    while (high - low > 1) {
        const int mid = low + (high - low) / 2;
        if (wave_sum_int(dearer(mid)) > t) low = mid;
        else high = mid;
    }
    // cost `high`: at most one item per sequence
    const bool has = base < high && high <= base + tiles;
    const uint64_t with = ballot(has);
    int nth = t - wave_sum_int(dearer(high));
    const uint64_t who = ballot(has && (int)lanes_below(with) == nth);
    if (who == 0) return {{-1, 0}, {0, 0}, {0, 0}};
    const int seq = __builtin_ctzll(who);
    auto of = [&](int v) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(v, seq); };
    return {{seq, high - 1 - of(base)}, {of(q.first), of(q.count)}, {of(k.first), of(k.count)}};
}

// Split keys.  A sequence's tiles of rows are each shared by `parts` workgroups, which take as many keys each
// as lets all workgroups together stay within `groups`: the longest sequences are split most, and no split is
// much longer than another.  Lane s has sequence s; `first` counts the workgroups of those before it.
struct Parts {
    int tiles, parts, first;
};
constexpr int kMinPart = 8;  // tiles of keys
__device__ __forceinline__ int key_tiles(const Rows& q, const Rows& k) { return q.count > 0 ? (k.count + kKeys - 1) / kKeys : 0; }
// Tiles of keys of a part.
__device__ __forceinline__ int part_length(const PackedArgs& A, const Rows& q, const Rows& k) {
    const int tiles = row_tiles(A, q.count), keys = key_tiles(q, k);
    int low = kMinPart - 1, high = max(wave_max_int(keys), kMinPart);  // high is long enough, low is not
    while (high - low > 1) {
        const int mid = low + (high - low) / 2;
        if (wave_sum_int(tiles * max((keys + mid - 1) / mid, 1)) <= A.groups) high = mid;
        else low = mid;
    }
    return high;
}
__device__ __forceinline__ Parts split_parts(const PackedArgs& A, const Rows& q, const Rows& k, int length) {
    const int tiles = row_tiles(A, q.count), parts = max((key_tiles(q, k) + length - 1) / length, 1);
    return {tiles, parts, wave_scan_int(tiles * parts) - tiles * parts};
}

template <bool SPLIT>
__global__ void __launch_bounds__(kThreads, 2) packed_kernel(PackedArgs A) {
    __shared__ __align__(16) uint16_t s_k[2][kKeys * kDim];
    __shared__ __align__(16) uint16_t s_v[2][kDim * kVPitch];
    __shared__ __align__(16) uint16_t s_out[kWaves][kWaveRows * kOutPitch];
    __shared__ int s_odd[2];  // the last tile on the diagonal whose V held a value that is not finite, per buffer
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, half = lane >> 5;
    // the KV heads take turns, so that a head's workgroups share an XCD's L2 when there are 8 heads
    int w = blockIdx.x;
    const int hk = w % A.Hk;
    w /= A.Hk;
    auto clear_rest = [&](int spare, int spares) __attribute__((always_inline)) {  // rows of no sequence
        const int begin = min(max(A.q_offsets[0], 0), A.Nq);
        const int end = min(max(A.q_offsets[A.sequences], begin), A.Nq);
        const int rest = begin + A.Nq - end;
        const int per_row = A.G * 16;  // 16-byte pieces of a query's heads in the group
        for (long i = (long)spare * kThreads + tid; i < (long)rest * per_row; i += (long)spares * kThreads) {
            const int r = (int)(i / per_row), at = (int)(i - (long)r * per_row);
            const long row = r < begin ? r : end + r - begin;
            reinterpret_cast<uint4*>(A.out + (row * A.Hq + (long)hk * A.G) * kDim)[at] = make_uint4(0, 0, 0, 0);
        }
    };
    Rows q_rows = {0, 0}, k_rows = {0, 0};  // of sequence `lane`
    if (A.sequences <= kWave && lane < A.sequences) {
        q_rows = sequence_rows(A.q_offsets, lane, A.Nq);
        k_rows = sequence_rows(A.k_offsets, lane, A.Nk);
    }
    Item it;
    Rows qr, kr;  // of the workgroup's sequence, kept in scalar registers
    int split = 0, parts = 1;
    if (SPLIT) {
        if (A.clear_rest) clear_rest(w, A.groups);
        const int length = part_length(A, q_rows, k_rows);
        if (blockIdx.x == 0 && tid == 0) *A.length = length;  // for the merge
        const Parts p = split_parts(A, q_rows, k_rows, length);
        const uint64_t who = ballot(w >= p.first && w < p.first + p.tiles * p.parts);
        if (who == 0) return;
        it.seq = __builtin_ctzll(who);
        parts = __builtin_amdgcn_readlane(p.parts, it.seq);
        const int n = w - __builtin_amdgcn_readlane(p.first, it.seq);
        it.index = n / parts;
        split = n - it.index * parts;
        qr = {__builtin_amdgcn_readlane(q_rows.first, it.seq), __builtin_amdgcn_readlane(q_rows.count, it.seq)};
        kr = {__builtin_amdgcn_readlane(k_rows.first, it.seq), __builtin_amdgcn_readlane(k_rows.count, it.seq)};
    } else {
        const Place place = A.sequences <= kWave ? place_by_cost(A, w, q_rows, k_rows) : place_in_order(A, w);
        it = place.item;
        if (it.seq < 0) {  // behind the last item (there is always one such)
            if (A.clear_rest) clear_rest(it.index, A.items - (w - it.index));
            return;
        }
        qr = place.q;
        kr = place.k;
    }
    const int nk = kr.count, ahead = nk - qr.count;          // query i sees keys up to i + ahead
    const int rows = qr.count * A.G, g0 = it.index * kRows;  // the sequence's rows, the workgroup's first
    const int r0 = g0 + wave * kWaveRows;                    // the wave's first row
    if (it.index < 0 || g0 >= rows) return;
    const int r = min(r0 + col, rows - 1);
    const int query = r / A.G, head = hk * A.G + r - query * A.G;
    const int sees = min(query + ahead + 1, nk);  // keys that this lane's row sees; none when not positive
    // keys that all rows of the wave see, and that some row sees; the same of the workgroup
    const int wave_all = min(r0, rows - 1) / A.G + ahead + 1;
    const int wave_any = r0 < rows ? min((min(r0 + kWaveRows, rows) - 1) / A.G + ahead + 1, nk) : 0;
    const int group_all = g0 / A.G + ahead + 1;
    const int group_any = min((min(g0 + kRows, rows) - 1) / A.G + ahead + 1, nk);
    const int tiles = group_any > 0 ? (group_any + kKeys - 1) / kKeys : 0;
    const int per_split = (tiles + parts - 1) / parts;
    const int tile0 = split * per_split, tile1 = min(tile0 + per_split, tiles);

    // Tiles are fetched through range-checked buffer loads without branches: a row behind the
    // sequence's last key lies behind the resource's end and comes as zeros.
    const int k_step = (int)A.k_token * 2, v_step = (int)A.v_token * 2;  // bytes
    const char* const v_base = (const char*)(A.v + kr.first * A.v_token + hk * A.v_head);
    // Each half of the workgroup brings one of the two, in 16-byte pieces.  K: thread (row = part / 16 + 16 i, place =
    // part % 16) brings piece place ^ row % 16; V: thread (keys 4 (part % 16) + i, piece = part / 16).
    const int part = tid & 255;
    const bool first = wave < 4;  // of the two halves
    const int step = first ? v_step : k_step;
    int at[4];  // the whole offset in the lane's: a scalar one would be left out of the range check
#pragma unroll
    for (int i = 0; i < 4; ++i)
        at[i] = first ? (4 * (part & 15) + i) * v_step + 16 * (part >> 4)
                      : (16 * i + (part >> 4)) * k_step + 16 * ((part & 15) ^ (part >> 4));
    const char* next = (first ? v_base : (const char*)(A.k + kr.first * A.k_token + hk * A.k_head)) + (long)tile0 * kKeys * step;
    int left = nk - tile0 * kKeys;  // rows from there on
    uint4 reg[4];
    auto fetch = [&]() __attribute__((always_inline)) {
        const __amdgpu_buffer_rsrc_t res = __builtin_amdgcn_make_buffer_rsrc(
            (void*)next, 0, left > 0 ? (min(left, kKeys) - 1) * step + 2 * kDim : 0, 0x00020000);
#pragma unroll
        for (int i = 0; i < 4; ++i) reg[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(res, at[i], 0, 0));
        next += (long)kKeys * step;
        left -= kKeys;
    };
    fetch();  // before Q, so that the first tile does not wait for it

    // Q operand: lane (col, half) holds its row, channels 16 kk + 8 half + [0, 8)
    half8_t qf[8];
    {
        const uint4* src = reinterpret_cast<const uint4*>(A.q + (qr.first + query) * A.q_token + head * A.q_head);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) qf[kk] = __builtin_bit_cast(half8_t, src[2 * kk + half]);
    }

    auto stage_k = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) reinterpret_cast<uint4*>(s_k[buf])[part + 256 * i] = reg[i];
    };
    // A key that a row does not see has weight 0, and its value must not matter to the row, also
    // when it is infinite or NaN: in the tiles on the diagonal such values are staged as zeros
    // and added to the rows that see them apart.
    auto stage_v = [&](int tile, int buf) __attribute__((always_inline)) {
        if ((tile + 1) * kKeys > group_all) {
            half2_t zero = {(_Float16)0.0f, (_Float16)0.0f}, sum = zero;  // NaN when a value is not finite
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t w[4] = {reg[i].x, reg[i].y, reg[i].z, reg[i].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) sum += __builtin_bit_cast(half2_t, w[e]) * zero;
            }
            if (!(sum[0] == 0.0f && sum[1] == 0.0f)) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    reg[i] = make_uint4(finite_or_zero(reg[i].x), finite_or_zero(reg[i].y), finite_or_zero(reg[i].z),
                                        finite_or_zero(reg[i].w));
                s_odd[buf] = tile;
            }
        }
        // four keys' 8 channels become 8 channels' four keys; key 4 q + i of a group of 16 goes to place 8 (q % 2) + 4 (q / 2) + i
        const int b = part & 15, q = b & 3;
        uint16_t* const dst = s_v[buf] + 8 * (part >> 4) * kVPitch + 16 * (b >> 2) + 8 * (q & 1) + 4 * (q >> 1);
        const uint32_t in[4][4] = {{reg[0].x, reg[0].y, reg[0].z, reg[0].w}, {reg[1].x, reg[1].y, reg[1].z, reg[1].w},
                                   {reg[2].x, reg[2].y, reg[2].z, reg[2].w}, {reg[3].x, reg[3].y, reg[3].z, reg[3].w}};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;  // the upper or lower halves of two dwords
            *reinterpret_cast<uint2*>(dst + e * kVPitch) =
                make_uint2(__builtin_amdgcn_perm(in[1][e >> 1], in[0][e >> 1], sel), __builtin_amdgcn_perm(in[3][e >> 1], in[2][e >> 1], sel));
        }
    };

    float16_t acc[4];  // O^T: channels 32 db + 8 (i / 4) + 4 half + i % 4 of the lane's row
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[db][i] = 0.0f;
    // log2-domain reference of the weights, and this lane's half of their sum.  The reference starts at
    // the lowest finite value: scores of minus infinity then weigh exp2(-inf) = 0, where
    // against a reference of minus infinity they would give NaN
    float m = -__FLT_MAX__, l = 0.0f;
    const half2_t ones = {(_Float16)1.0f, (_Float16)1.0f};
    // K operand: piece 2 kk + half of row col (and 32 + col, permuted alike) lies at place (2 kk + half) ^ col % 16
    const int k_read = col * 2 * kDim + 16 * (half ^ (col & 15));  // bytes, of kk = 0

    float16_t s[2];
    auto scores = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[kb][i] = 0.0f;
#pragma unroll
            for (int kk = 0; kk < 8; ++kk) {
                const half8_t kf = *reinterpret_cast<const half8_t*>((const char*)s_k[buf] + 64 * kb * kDim + (k_read ^ 32 * kk));
                s[kb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[kk], s[kb], 0, 0, 0);
            }
        }
        // reads ahead of the products by four
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
        for (int i = 0; i < 12; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
    };
    auto values = [&](int tile, int buf) __attribute__((always_inline)) {
        if ((tile + 1) * kKeys > wave_all) {  // the diagonal
            const int seen = sees - tile * kKeys - 4 * half;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (32 * kb + 8 * (i >> 2) + (i & 3) >= seen) s[kb][i] = -INFINITY;
        }
        float mx = s[0][0];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[kb][i]);
        const auto sw = __builtin_amdgcn_permlane32_swap((uint32_t)f2i(mx), (uint32_t)f2i(mx), false, false);
        mx = fmaxf(i2f((int)sw[0]), i2f((int)sw[1])) * A.c;  // c > 0
        if (ballot(mx > m + kSlack) != 0) {
            const float mn = fmaxf(m, mx);
            const float alpha = __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int db = 0; db < 4; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[db][i] *= alpha;
        }
        const float shift = kWeightBits - m;
        float sum = 0.0f;  // of the tile: each pair of weights added to l itself would be rounded against a large sum
        const uint16_t* const sv = s_v[buf] + col * kVPitch + 8 * half;
#pragma unroll
        for (int st = 0; st < 4; ++st) {
            half8_t pf;  // the weights of a 16-key step, keys in the lane's order
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const half2_t p = {(_Float16)__builtin_amdgcn_exp2f(__builtin_fmaf(s[st >> 1][8 * (st & 1) + i], A.c, shift)),
                                   (_Float16)__builtin_amdgcn_exp2f(__builtin_fmaf(s[st >> 1][8 * (st & 1) + i + 1], A.c, shift))};
                sum = __builtin_amdgcn_fdot2(p, ones, sum, false);
                pf[i] = p[0];
                pf[i + 1] = p[1];
            }
#pragma unroll
            for (int db = 0; db < 4; ++db) {
                const half8_t vf = *reinterpret_cast<const half8_t*>(sv + 32 * db * kVPitch + 16 * st);
                acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pf, acc[db], 0, 0, 0);
            }
        }
        l += sum;
        // a step's weights between the products of the step before
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
        for (int i = 0; i < 12; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
        if ((tile + 1) * kKeys > group_all && s_odd[buf] == tile) {  // rare: what was staged as zero, to the rows that see it
            const int last = min((tile + 1) * kKeys, nk);
            for (int j = tile * kKeys; j < last; ++j) {
                const uint16_t* row = (const uint16_t*)(v_base + (long)j * v_step);
#pragma unroll
                for (int db = 0; db < 4; ++db)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float x = h2f(row[32 * db + 8 * (i >> 2) + 4 * half + (i & 3)]);
                        if (j < sees && !(fabsf(x) < INFINITY)) acc[db][i] += x;
                    }
            }
        }
    };

    // The halves take turns: while one multiplies with K, the other does its softmax and multiplies with V, half a
    // tile behind.  Each brings its share of the next tile in the first of these.
    if (tid < 2) s_odd[tid] = -1;
    if (!first) {
        stage_k(0);
        fetch();
    }
    __syncthreads();
    // (both halves meet 2 n + 1 barriers for n tiles: the second one starts a barrier later and needs none
    // behind its last tile)
    if (!first && tile0 < tile1) __syncthreads();
    for (int tile = tile0; tile < tile1; ++tile) {
        const int buf = (tile - tile0) & 1;
        const bool sees_any = tile * kKeys < wave_any;  // wave-uniform: a tile that no row of the wave sees is left out
        if (first) stage_v(tile, buf);
        else stage_k(buf ^ 1);
        fetch();
        if (sees_any) scores(buf);
        __syncthreads();
        if (sees_any) values(tile, buf);
        if (first || tile + 1 < tile1) __syncthreads();
    }
    const auto ls = __builtin_amdgcn_permlane32_swap((uint32_t)f2i(l), (uint32_t)f2i(l), false, false);
    const float total = i2f((int)ls[0]) + i2f((int)ls[1]);
    if (SPLIT && parts > 1) {
        if (r0 + col >= rows) return;
        const long record = (long)blockIdx.x * A.record_rows + wave * kWaveRows + col;
        float* rec = A.part + record * kDim;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int i = 0; i < 16; i += 2)
                *reinterpret_cast<float2*>(rec + 32 * db + 8 * (i >> 2) + 4 * half + (i & 3)) = make_float2(acc[db][i], acc[db][i + 1]);
        if (half == 0) A.stat[record] = make_float2(m, total);
        return;
    }
    // through the LDS to whole rows: sixteen lanes write one
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    uint16_t* const mine = s_out[wave];
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t word[2];
#pragma unroll
            for (int e = 0; e < 2; ++e)
                word[e] = (uint32_t)f2h(acc[db][4 * j + 2 * e] * inv) | ((uint32_t)f2h(acc[db][4 * j + 2 * e + 1] * inv) << 16);
            *reinterpret_cast<uint2*>(mine + col * kOutPitch + 32 * db + 8 * j + 4 * half) = make_uint2(word[0], word[1]);
        }
    wave_sync();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int n = 4 * i + (lane >> 4), at_row = r0 + n;
        if (at_row >= rows) break;
        const int of = at_row / A.G;
        reinterpret_cast<uint4*>(A.out + (((long)qr.first + of) * A.Hq + hk * A.G + at_row - of * A.G) * kDim)[lane & 15] =
            *reinterpret_cast<const uint4*>(mine + n * kOutPitch + 8 * (lane & 15));
    }
}

// Joins the splits: two (query, head) rows per wave, four channels per lane, eight records of a row at a time
// under a running maximum, so that a row costs two trips to memory (offsets, records).  Rows of no sequence, and
// of sequences that are not split, are done already.  One row at a time with the maximum of all its records first
// cost 4 us more (3 chunks of 33 to 200 tokens after 20000: 125.6 us for both kernels against 121.7).
constexpr int kMergeRows = 2;  // a half of the wave each
__global__ void __launch_bounds__(kThreads) packed_merge_kernel(PackedArgs A) {
    const int lane = threadIdx.x & 63;
    const long row0 = ((long)blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * kMergeRows;
    if (row0 >= (long)A.Nq * A.Hq) return;
    Rows q = {0, 0}, k = {0, 0};
    if (lane < A.sequences) {
        q = sequence_rows(A.q_offsets, lane, A.Nq);
        k = sequence_rows(A.k_offsets, lane, A.Nk);
    }
    const Parts p = split_parts(A, q, k, *A.length);
    const int half = lane >> 5;
    int parts = 1, group = 0, r = 0, most_parts = 1;  // of the lane's row
#pragma unroll
    for (int h = 0; h < kMergeRows; ++h) {
        const int query = (int)((row0 + h) / A.Hq);
        const uint64_t who = ballot(query < A.Nq && query >= q.first && query < q.first + q.count);
        if (who == 0) continue;
        const int seq = __builtin_ctzll(who), n = __builtin_amdgcn_readlane(p.parts, seq);
        const int head = (int)(row0 + h - (long)query * A.Hq);
        const int at = (query - __builtin_amdgcn_readlane(q.first, seq)) * A.G + head % A.G;
        const int g = __builtin_amdgcn_readlane(p.first, seq) + at / kRows * n;
        if (n == 1 || g + n > A.groups) continue;
        most_parts = max(most_parts, n);
        if (half == h) {
            parts = n;
            // workgroup (first + tile * parts + split) * Hk + hk has the row's record of a split
            group = g * A.Hk + head / A.G;
            r = at % kRows;
        }
    }
    if (most_parts == 1) return;
    const long record = (long)group * A.record_rows + r, apart = (long)A.Hk * A.record_rows;
    const float4* const rec = reinterpret_cast<const float4*>(A.part) + record * 32 + (lane & 31);
    float top = -__FLT_MAX__, o0 = 0.0f, o1 = 0.0f, o2 = 0.0f, o3 = 0.0f, total = 0.0f;
    for (int s0 = 0; s0 < most_parts; s0 += 8) {
        float4 o[8];
        float2 ml[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const long at = min(s0 + j, parts - 1) * apart;
            o[j] = rec[at * 32];
            ml[j] = A.stat[record + at];
        }
        float most = top;
#pragma unroll
        for (int j = 0; j < 8; ++j) most = fmaxf(most, ml[j].x);
        const float alpha = __builtin_amdgcn_exp2f(top - most);
        o0 *= alpha, o1 *= alpha, o2 *= alpha, o3 *= alpha, total *= alpha;
        top = most;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (s0 + j >= parts || ml[j].y == 0.0f) continue;  // no keys (a NaN goes on)
            const float a = __builtin_amdgcn_exp2f(ml[j].x - top);
            o0 += a * o[j].x;
            o1 += a * o[j].y;
            o2 += a * o[j].z;
            o3 += a * o[j].w;
            total += a * ml[j].y;
        }
    }
    if (parts == 1) return;
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    reinterpret_cast<uint2*>(A.out + (row0 + half) * kDim)[lane & 31] =
        make_uint2((uint32_t)f2h(o0 * inv) | ((uint32_t)f2h(o1 * inv) << 16), (uint32_t)f2h(o2 * inv) | ((uint32_t)f2h(o3 * inv) << 16));
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

// Tiles of 256 rows that S sequences of Nq rows in all can bring, and one that is always free.
long packed_items(int S, long Nq, int G) { return Nq * G / kRows + S + 1; }

// Whether the keys are split: while the rows alone leave CUs without a workgroup and there are keys for more
// than one part.  Workgroups of a KV head then (one per CU in all), else 0.  Where the keys are mostly
// the queries' own, the tiles differ in length and the longest of them bounds the time less than a second
// pass over the records costs, so that half of the CUs have to be free: one prompt of 1600 tokens (200 workgroups)
// 50 us whole and 73 split; 20 chunks of 10 tokens after 5000 (160 workgroups) 86 whole and 71 split.
constexpr int kGroups = 256;
int split_groups(int S, long Nq, int Hk, int G, long max_keys) {
    const long groups = packed_items(S, Nq, G) * Hk * (max_keys < 4 * Nq ? 2 : 1);
    return S <= kWave && groups <= kGroups && max_keys >= 2 * kMinPart * kKeys ? kGroups / Hk : 0;
}

// Rows of a workgroup that can hold a record: no sequence has more than all rows.
long record_rows(long Nq, int G) { return Nq * G < kRows ? Nq * G : kRows; }

}  // namespace

extern "C" int64_t reskv_packed_workspace_bytes(int S, int64_t Nq, int Hq, int Hk, int64_t max_keys) {
    if (S < 1 || Nq < 1 || Hk < 1 || Hq < 1 || Hq % Hk != 0 || Nq >= (1LL << 30)) return 0;
    const int64_t groups = split_groups(S, Nq, Hk, Hq / Hk, max_keys);
    return groups == 0 ? 0 : groups * Hk * record_rows(Nq, Hq / Hk) * kRecord * 4 + 16;  // records, length of a part
}

extern "C" int reskv_packed_attention(const void* q, const void* k, const void* v, void* out, const int32_t* q_offsets,
                                      const int32_t* k_offsets, int S, int64_t Nq, int64_t Nk, int Hq, int Hk,
                                      const int64_t* strides, float scaling, int64_t max_keys, int clear_rest,
                                      void* workspace, int64_t workspace_bytes, void* stream) {
    RESKV_REQUIRE(q && k && v && out && q_offsets && k_offsets && strides, "null pointer");
    RESKV_REQUIRE(S > 0 && Nq > 0 && Nk > 0 && Hk > 0 && Hq > 0 && Hq % Hk == 0,
                  "bad sizes (sequences %d, Nq %ld, Nk %ld, Hq %d, Hk %d)", S, (long)Nq, (long)Nk, Hq, Hk);
    const int G = Hq / Hk;
    RESKV_REQUIRE(Nq * G < (1LL << 30) && Nk < (1LL << 30), "too many rows");
    RESKV_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out) && aligned16(workspace), "tensors must be 16-byte aligned");
    for (int i = 0; i < 6; ++i) RESKV_REQUIRE(strides[i] >= 0 && strides[i] % 8 == 0, "rows must be 16-byte aligned");
    RESKV_REQUIRE(strides[2] < (1 << 23) && strides[4] < (1 << 23), "token strides of k and v must be below 2^23");
    RESKV_REQUIRE(strides[2] >= kDim && strides[4] >= kDim, "rows of k and v must not overlap");
    RESKV_REQUIRE(scaling > 0.0f && scaling < 1e30f, "scaling must be positive and below 1e30");
    const int split = split_groups(S, Nq, Hk, G, max_keys);
    RESKV_REQUIRE(!split || (workspace && workspace_bytes >= reskv_packed_workspace_bytes(S, Nq, Hq, Hk, max_keys)),
                  "the workspace is too small");
    PackedArgs A{};
    A.q = (const uint16_t*)q;
    A.k = (const uint16_t*)k;
    A.v = (const uint16_t*)v;
    A.out = (uint16_t*)out;
    A.q_offsets = q_offsets;
    A.k_offsets = k_offsets;
    A.part = (float*)workspace;
    A.record_rows = (int)record_rows(Nq, G);
    A.stat = (float2*)(A.part + (long)split * Hk * A.record_rows * kDim);
    A.length = (int32_t*)(A.stat + (long)split * Hk * A.record_rows);
    A.q_token = strides[0];
    A.q_head = strides[1];
    A.k_token = strides[2];
    A.k_head = strides[3];
    A.v_token = strides[4];
    A.v_head = strides[5];
    A.sequences = S;
    A.Nq = (int)Nq;
    A.Nk = (int)Nk;
    A.Hq = Hq;
    A.Hk = Hk;
    A.G = G;
    const long items = packed_items(S, Nq, G);
    RESKV_REQUIRE(items * Hk < kLaunchThreads / kThreads, "too many rows or sequences");
    A.items = (int)items;
    A.groups = split;
    A.clear_rest = clear_rest;
    A.c = scaling * 1.4426950408889634f;
    hipLaunchKernelGGL(split ? packed_kernel<true> : packed_kernel<false>, dim3((unsigned)(split ? split * Hk : items * Hk)),
                       dim3(kThreads), 0, (hipStream_t)stream, A);
    if (reskv_host::check_launch("packed_kernel")) return 1;
    if (!split) return 0;
    const long rows = (long)Nq * Hq;
    hipLaunchKernelGGL(packed_merge_kernel, dim3((unsigned)((rows + kWaves * kMergeRows - 1) / (kWaves * kMergeRows))), dim3(kThreads), 0,
                       (hipStream_t)stream, A);
    return reskv_host::check_launch("packed_merge_kernel");
}
