// Trees of drafted tokens (include/reskv_drafts.h): their masks, which of them the target model accepts, and the pages'
// tokens of those moved together.
#include "int4.h"
#include "reskv_drafts.h"

using namespace reskv;

namespace {

constexpr int kNodes = RESKV_DRAFT_NODES;  // one per lane

// ---------------------------------------------------------------------------
// masks and positions
// ---------------------------------------------------------------------------

// One wave per sequence, a lane per node.  A node's ancestors by doubling: the mask of its parent joins its own and its parent
// becomes its parent's parent, six times for 64 nodes.
__global__ void __launch_bounds__(kWave) tree_masks_kernel(const int32_t* parents, const int32_t* offsets, const int32_t* starts, int N,
                                                           uint64_t* seen, int32_t* positions) {
    const Rows r = sequence_rows(offsets, (int)blockIdx.x, N);
    const int lane = threadIdx.x, n = min(r.count, kNodes);
    int up = lane < n ? parents[r.first + lane] : -1;
    if (up >= lane || up < 0) up = lane;  // a root is its own parent
    uint64_t mask = 1ull << lane;
#pragma unroll
    for (int i = 0; i < 6; ++i) {
        const uint32_t low = __shfl((int)(uint32_t)mask, up), high = __shfl((int)(uint32_t)(mask >> 32), up);
        up = __shfl(up, up);
        mask |= (uint64_t)high << 32 | low;
    }
    if (lane >= n) return;
    seen[r.first + lane] = mask;
    if (positions) positions[r.first + lane] = (starts ? starts[blockIdx.x] : 0) + __popcll(mask) - 1;
}

// ---------------------------------------------------------------------------
// verification
// ---------------------------------------------------------------------------

constexpr int kSegments = 64;         // of a row, at most: one per lane
constexpr int kPiece = 8;             // elements that a thread takes at once
constexpr double kSmall = 0x1p-20;    // of a row's or a segment's sum: what is left of less is added up anew, as a difference has lost its bits
constexpr int kStatThreads = 256;
// Of a walk: greedy, 16 waves take the statistics of 64 rows (24 trees 36 us in all, 38 with eight); else every barrier counts (32
// chains with draft probabilities 33 us with eight waves, 37 with 16, 38 with four).
constexpr int walk_threads(bool greedy) { return greedy ? 1024 : 512; }

// A walk that waits for the sums of what a draft that was turned down leaves.
struct WalkState {
    double left;       // sum of r before it
    int here, length, down;  // the node reached, the path so far, the draft; down 0: the walk is at its end
};

struct VerifyArgs {
    const void* logits;
    const int64_t* tokens;
    const int32_t *parents, *offsets;
    const float *accept, *sample, *draft;
    long row_stride, draft_stride, V;
    int32_t *path, *counts;
    int64_t* token;
    double* sum;       // [N, segments]: of exp2((x - most) c)
    float* most;       // [N, segments]
    int32_t* arg;      // [N, segments], temperature 0: where the maximum is, -1 where there is a NaN
    double* rest;      // [S, segments], with draft: what the first draft turned down leaves of r
    WalkState* state;  // [S], with draft: where the walk stands there
    double c;          // log2(e) / temperature
    int N, segments, pieces;  // pieces of a segment
};

// 2^y for -2000 <= y <= 0, to 2^-38 of itself: the series of 2^f for a fraction f of at most a half (its coefficients are ln(2)^k /
// k!), from the fifth power on, where it is below 2^-14, in 32 bits.  A NaN goes on.
__device__ __forceinline__ double exp2_of(double y) {
    constexpr double l = 0.69314718055994530942, l2 = l * l, l4 = l2 * l2, l8 = l4 * l4;
    const double whole = __builtin_rint(y), f = y - whole;
    const float g = (float)f;
    float tail = (float)(l8 * l2 / 3628800.0);
    tail = __builtin_fmaf(tail, g, (float)(l8 * l / 362880.0));
    tail = __builtin_fmaf(tail, g, (float)(l8 / 40320.0));
    tail = __builtin_fmaf(tail, g, (float)(l4 * l2 * l / 5040.0));
    tail = __builtin_fmaf(tail, g, (float)(l4 * l2 / 720.0));
    tail = __builtin_fmaf(tail, g, (float)(l4 * l / 120.0));
    double p = __builtin_fma((double)tail, f, l4 / 24.0);
    p = __builtin_fma(p, f, l2 * l / 6.0);
    p = __builtin_fma(p, f, l2 / 2.0);
    p = __builtin_fma(p, f, l);
    p = __builtin_fma(p, f, 1.0);
    return __builtin_ldexp(p, (int)whole);  // 0 where it is below 2^-1074
}
// The weight of a logit x against the largest, without a branch: 0 for minus infinity, also where there is nothing else.
__device__ __forceinline__ double weight_of(float x, float most, double c) {
    const double y = ((double)x - (double)fmaxf(most, -__FLT_MAX__)) * c;
    return exp2_of(y < -2000.0 ? -2000.0 : y);
}

template <class T>
__device__ __forceinline__ float element(const T* p) { return *p; }
template <>
__device__ __forceinline__ float element<uint16_t>(const uint16_t* p) { return h2f(*p); }

// Elements 8 p - shift .. + 7 of a row, whose pieces are 16 bytes of aligned fp16 memory (or twice that of fp32); minus infinity for
// those that are not in the row.  `fetch` reads without a branch, a piece inside the row where p is not.
template <class T>
struct Row {
    static constexpr int kWords = sizeof(T) / 2;
    struct Raw {
        uint4 w[kWords];
    };
    const T* p;
    long V;
    int shift, full0, full1;  // the pieces that are wholly inside
    __device__ __forceinline__ Row(const VerifyArgs& A, int row)
        : p((const T*)A.logits + row * A.row_stride), V(A.V), shift((int)(((uintptr_t)p & 15) / sizeof(T))) {
        full0 = shift > 0 ? 1 : 0;
        full1 = (int)((V + shift) / kPiece) - 1;
    }
    __device__ __forceinline__ int pieces() const { return (int)((V + shift + kPiece - 1) / kPiece); }
    __device__ __forceinline__ long first(int piece) const { return (long)piece * kPiece - shift; }
    __device__ __forceinline__ void fetch(int piece, Raw& raw) const {
        if (full1 < full0) return;  // (the same for every thread)
        const uint4* const src = reinterpret_cast<const uint4*>(p + first(min(max(piece, full0), full1)));
#pragma unroll
        for (int i = 0; i < kWords; ++i) raw.w[i] = src[i];
    }
    __device__ __forceinline__ void values(int piece, int end, const Raw& raw, float* x) const {
        const uint4 w0 = raw.w[0], w1 = raw.w[kWords - 1];
        const uint32_t d[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
        for (int i = 0; i < kPiece; ++i) x[i] = sizeof(T) == 2 ? h2f((uint16_t)(d[i >> 1] >> (16 * (i & 1)))) : i2f((int)d[i]);
        if (piece >= full0 && piece <= full1 && piece < end) return;
        const long at = first(piece);
#pragma unroll
        for (int i = 0; i < kPiece; ++i) x[i] = piece < end && at + i >= 0 && at + i < V ? element(p + at + i) : -INFINITY;
    }
    __device__ __forceinline__ void load(int piece, int end, float* x) const {
        Raw raw;
        fetch(piece, raw);
        values(piece, end, raw, x);
    }
};

template <int CTRL>
__device__ __forceinline__ double dpp_double(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)dpp_u<CTRL>((uint32_t)(b >> 32)) << 32 | dpp_u<CTRL>((uint32_t)b));
}
__device__ __forceinline__ double lane_double(double v, int lane) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(b >> 32), lane) << 32 |
                                          (uint32_t)__builtin_amdgcn_readlane((int)b, lane));
}
__device__ __forceinline__ double wave_sum_double(double v) {
    v += dpp_double<0xB1>(v);
    v += dpp_double<0x4E>(v);
    v += dpp_double<0x141>(v);
    v += dpp_double<0x140>(v);
    return (lane_double(v, 0) + lane_double(v, 16)) + (lane_double(v, 32) + lane_double(v, 48));
}
// Inclusive sums in lane order.
__device__ __forceinline__ double wave_scan_double(double v, int lane) {
#pragma unroll
    for (int i = 1; i < kWave; i *= 2) {
        const double other = __shfl_up(v, i);
        if (lane >= i) v += other;
    }
    return v;
}

// Each row's segments: the largest logit and the sum of exp2((x - largest) c) in 64 bits, or where the largest is.  A thread
// keeps its own maximum and brings its sum down when that moves; PIECES of them are under way at once.
//
// Bound: greedy by memory (558 rows of 128256: 32 us, 4.5 TB/s), else by the 64-bit exponentials (192 rows of 32003: 10 us, where
// the bytes alone would take 2.6; 14 with a branch per element and the series in 64 bits throughout).  In 32 bits the sums would turn a
// sampled token now and then: a token's share of a wide vocabulary is 1e-5 and less.
template <class T, bool GREEDY, int PIECES>
__global__ void __launch_bounds__(kStatThreads) verify_stat_kernel(VerifyArgs A) {
    __shared__ float s_most[kStatThreads / kWave];
    __shared__ double s_sum[kStatThreads / kWave];
    __shared__ int s_arg[kStatThreads / kWave];
    const int row = (int)(blockIdx.x / A.segments), segment = (int)(blockIdx.x - (long)row * A.segments);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const Row<T> R(A, row);
    const int last = min((segment + 1) * A.pieces, R.pieces());
    float most = -INFINITY;
    double sum = 0.0;
    int arg = 0x7FFFFFFF;
    bool nan = false;
    for (int p0 = segment * A.pieces + tid; p0 < last; p0 += PIECES * kStatThreads) {
        typename Row<T>::Raw raw[PIECES];
#pragma unroll
        for (int k = 0; k < PIECES; ++k) R.fetch(p0 + k * kStatThreads, raw[k]);
        float x[PIECES][kPiece];
#pragma unroll
        for (int k = 0; k < PIECES; ++k) R.values(p0 + k * kStatThreads, last, raw[k], x[k]);
        if (GREEDY) {
#pragma unroll
            for (int k = 0; k < PIECES; ++k)
#pragma unroll
                for (int i = 0; i < kPiece; ++i) {
                    const int p = p0 + k * kStatThreads;
                    const long at = R.first(p) + i;
                    nan |= x[k][i] != x[k][i];
                    if (p < last && at >= 0 && at < A.V && (x[k][i] > most || arg == 0x7FFFFFFF)) {
                        most = x[k][i];
                        arg = (int)at;
                    }
                }
        } else {
            float top = x[0][0];
#pragma unroll
            for (int i = 1; i < PIECES * kPiece; ++i) top = fmaxf(top, x[i / kPiece][i % kPiece]);
            if (top > most) {
                sum *= weight_of(most, top, A.c);
                most = top;
            }
#pragma unroll
            for (int i = 0; i < PIECES * kPiece; ++i) sum += weight_of(x[i / kPiece][i % kPiece], most, A.c);
        }
    }
    const float wave_most = wave_max(most);
    if (GREEDY) {
        // the first thread's in order of index among those that have the maximum
        int at = most == wave_most || arg == 0x7FFFFFFF ? arg : 0x7FFFFFFF;
#pragma unroll
        for (int i = 1; i < kWave; i *= 2) at = min(at, __shfl_xor(at, i));
        if (ballot(nan) != 0) at = -1;
        if (lane == 0) s_arg[wave] = at;
    } else {
        sum = most == wave_most || sum == 0.0 ? sum : sum * weight_of(most, wave_most, A.c);
        sum = wave_sum_double(sum);
        if (lane == 0) s_sum[wave] = sum;
    }
    if (lane == 0) s_most[wave] = wave_most;
    __syncthreads();
    if (tid != 0) return;
    const long at = (long)row * A.segments + segment;
    float top = s_most[0];
#pragma unroll
    for (int w = 1; w < kStatThreads / kWave; ++w) top = fmaxf(top, s_most[w]);
    A.most[at] = top;
    if (GREEDY) {
        int best = 0x7FFFFFFF;
        bool bad = false;
#pragma unroll
        for (int w = 0; w < kStatThreads / kWave; ++w) {
            bad |= s_arg[w] == -1;
            if (s_most[w] == top) best = min(best, s_arg[w]);
        }
        A.arg[at] = bad ? -1 : best;
    } else {
        double all = 0.0;
#pragma unroll
        for (int w = 0; w < kStatThreads / kWave; ++w)
            all += s_most[w] == top || s_sum[w] == 0.0 ? s_sum[w] : s_sum[w] * weight_of(s_most[w], top, A.c);
        A.sum[at] = all;
    }
}

// What the distribution q of a draft that was turned down leaves of a weight; scale is one over the sum of r.
__device__ __forceinline__ double less(double w, double scale, float q) {
    const double rest = w * scale - (double)q;
    return rest > 0.0 ? rest : 0.0;
}

// The walk down a tree, one workgroup per sequence.  Everything that the decisions need comes in one trip to memory, a lane
// per node: the node's token, its logit behind its parent, its draft probability, and its row's statistics from the
// segments.  The token at the end costs a pass over one segment.  A draft that was turned down costs, with `draft`, a pass
// over its row and the target's: the first one's is left to verify_rest_kernel, which has a workgroup per segment, and the walk
// goes on in a second launch (RESUME); any further ones (siblings that were drawn) are done by the workgroup alone.
//
// Bound: trips to memory and barriers (8 nodes 8 us, 24 greedy trees of up to 64 nodes 6).  The pass over a row by the walk's own
// workgroup made 32 chains of a vocabulary of 32003 55 us, where the four kernels now take 35.
template <class T, bool GREEDY, bool RESUME>
__global__ void __launch_bounds__(walk_threads(GREEDY)) verify_walk_kernel(VerifyArgs A) {
    constexpr int kWalkThreads = walk_threads(GREEDY), kWalkWaves = kWalkThreads / kWave;
    __shared__ double s_total[kNodes];  // of a node's row: sum of exp2((x - most) c)
    __shared__ float s_most[kNodes], s_logit[kNodes], s_q[kNodes], s_accept[kNodes];
    __shared__ int s_parent[kNodes], s_token[kNodes], s_best[kNodes], s_path[kNodes];
    __shared__ double s_segment[kSegments];              // what is left of r, by segment
    __shared__ double s_scan[kWalkWaves], s_part[kSegments][kWalkWaves];
    __shared__ int s_down[kNodes];                       // drafts turned down at the node reached: their nodes,
    __shared__ double s_scale[kNodes];                   // and one over the sum of r before them
    __shared__ int s_past[kWalkWaves], s_some[kWalkWaves];
    const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    WalkState W = {};
    if (RESUME) {
        W = A.state[s];
        if (W.down == 0) return;
    }
    const Rows rows = sequence_rows(A.offsets, s, A.N);
    const int n = min(rows.count, kNodes);
    if (n == 0) {
        if (tid < kNodes) A.path[(long)s * kNodes + tid] = -1;
        if (tid == 0) {
            A.counts[s] = 0;
            A.token[s] = -1;
            if (!GREEDY && A.draft) A.state[s].down = 0;
        }
        return;
    }
    const T* const logits = (const T*)A.logits + rows.first * A.row_stride;
    if (tid < n) {
        const int parent = A.parents[rows.first + tid];
        const int64_t t = A.tokens[rows.first + tid];
        const bool good = tid > 0 && parent >= 0 && parent < tid && t >= 0 && t < A.V;
        s_parent[tid] = good ? parent : -1;
        s_token[tid] = good ? (int)t : -1;
        if (!GREEDY && good) {
            s_logit[tid] = element(logits + parent * A.row_stride + t);
            s_q[tid] = A.draft ? A.draft[(rows.first + tid) * A.draft_stride + t] : 1.0f;
            s_accept[tid] = A.accept[rows.first + tid];
        }
        if (RESUME) s_path[tid] = A.path[(long)s * kNodes + tid];
    }
    for (int i = wave; i < n; i += kWalkWaves) {
        const long at = (long)(rows.first + i) * A.segments + lane;
        const bool in = lane < A.segments;
        const float most = in ? A.most[at] : -INFINITY;
        if (GREEDY) {
            const int arg = in ? A.arg[at] : 0x7FFFFFFF;
            const float top = wave_max(most);
            int best = most == top || arg == -1 ? arg : 0x7FFFFFFF;
#pragma unroll
            for (int j = 1; j < kWave; j *= 2) best = min(best, __shfl_xor(best, j));
            if (lane == 0) s_best[i] = best;
        } else {
            double sum = in ? A.sum[at] : 0.0;
            const float top = wave_max(most);
            if (sum != 0.0 && most != top) sum *= weight_of(most, top, A.c);
            sum = wave_sum_double(sum);
            if (lane == 0) {
                s_total[i] = sum;
                s_most[i] = top;
            }
        }
    }
    if (RESUME && tid < A.segments) s_segment[tid] = A.rest[(long)s * A.segments + tid];
    if (RESUME && tid == 0) {
        s_down[0] = W.down;
        s_scale[0] = 1.0 / W.left;
    }
    __syncthreads();

    const int parent = lane < n ? s_parent[lane] : -1, token = lane < n ? s_token[lane] : -1;
    int here = RESUME ? W.here : 0, length = RESUME ? W.length : 1;
    if (tid == 0) s_path[0] = 0;
    if (GREEDY) {
        while (const uint64_t child = ballot(parent == here && token == s_best[here])) {
            here = __builtin_ctzll(child);
            if (tid == 0) s_path[length] = here;
            ++length;
        }
        __syncthreads();
        if (tid < kNodes) A.path[(long)s * kNodes + tid] = tid < length ? s_path[tid] : -1;
        if (tid == 0) {
            A.counts[s] = length;
            A.token[s] = s_best[here];
        }
        return;
    }

    int down = 0;       // drafts turned down here
    double left = 0.0;  // sum of r
    bool whole = true;  // s_segment is not made yet: r is the softmax but for single tokens
    // r of an element of the row reached: its weight, without the tokens turned down, or with the drafts' distributions taken away
    auto weight = [&](float x, long at) __attribute__((always_inline)) {
        double w = weight_of(x, s_most[here], A.c);
        for (int i = 0; i < down; ++i) {
            if (A.draft) w = less(w, s_scale[i], A.draft[(rows.first + s_down[i]) * A.draft_stride + at]);
            else if (s_token[s_down[i]] == at) w = 0.0;
        }
        return w;
    };
    auto sum_segments = [&]() __attribute__((always_inline)) { return wave_sum_double(lane < A.segments ? s_segment[lane] : 0.0); };
    // The sums of r of segments g0 .. g1 - 1; returns that of all.
    auto measure = [&](int g0, int g1) __attribute__((always_inline)) {
        const Row<T> R(A, rows.first + here);
        for (int g = g0; g < g1; ++g) {
            const int last = min((g + 1) * A.pieces, R.pieces());
            double sum = 0.0;
            for (int p = g * A.pieces + tid; p < last; p += kWalkThreads) {
                float x[kPiece];
                R.load(p, last, x);
#pragma unroll
                for (int i = 0; i < kPiece; ++i)
                    if (!(x[i] == -INFINITY)) sum += weight(x[i], R.first(p) + i);
            }
            sum = wave_sum_double(sum);
            if (lane == 0) s_part[g][wave] = sum;
        }
        __syncthreads();
        if (tid >= g0 && tid < g1) {
            double sum = 0.0;
#pragma unroll
            for (int v = 0; v < kWalkWaves; ++v) sum += s_part[tid][v];
            s_segment[tid] = sum;
        }
        __syncthreads();
        return sum_segments();
    };
    uint64_t asked = ~0ull;  // nodes that are still to be looked at
    left = s_total[here];
    if (RESUME) {
        const double rest = sum_segments();
        if (rest > 0.0) {
            left = rest;
            down = 1;
            whole = false;
        }
        asked = ~((2ull << W.down) - 1);
    }
    while (left > 0.0 && left < INFINITY) {
        const uint64_t children = ballot(parent == here) & asked;
        if (children == 0) break;
        const int i = __builtin_ctzll(children);
        asked = ~((2ull << i) - 1);
        const int t = __builtin_amdgcn_readlane(token, i);
        const double w = weight(s_logit[i], t);
        if ((double)s_accept[i] * (double)s_q[i] < w / left) {
            here = i;
            if (tid == 0) s_path[length] = i;
            ++length;
            down = 0;
            whole = true;
            left = s_total[i];
            continue;
        }
        if (!A.draft && w == 0.0) continue;  // nothing to take away
        if (A.draft && !RESUME) {  // the sums of what is left come from the whole chip
            __syncthreads();
            if (tid < kNodes) A.path[(long)s * kNodes + tid] = tid < length ? s_path[tid] : -1;
            if (tid == 0) A.state[s] = {left, here, length, i};
            return;
        }
        __syncthreads();
        if (tid == 0) {
            s_down[down] = i;
            s_scale[down] = 1.0 / left;
        }
        __syncthreads();
        ++down;
        // without a distribution only one token goes; where that is nearly all, the rest is added up anew
        double rest = left - w;
        if (A.draft || !whole || !(rest > kSmall * s_total[here])) {
            rest = measure(0, A.segments);
            whole = false;
        }
        if (rest > 0.0) {
            left = rest;
        } else {
            --down;  // nothing left: r stays
            whole = true;
        }
    }
    __syncthreads();
    if (tid < kNodes) A.path[(long)s * kNodes + tid] = tid < length ? s_path[tid] : -1;
    if (tid == 0) {
        A.counts[s] = length;
        if (A.draft && !RESUME) A.state[s].down = 0;
    }
    if (!(left > 0.0 && left < INFINITY)) {
        if (tid == 0) A.token[s] = -1;
        return;
    }
    const Row<T> R(A, rows.first + here);
    if (whole) {
        if ((A.draft && down > 0) || !(left > kSmall * s_total[here])) {
            measure(0, A.segments);
        } else {
            // from the row's statistics, without the tokens turned down
            if (tid < A.segments) {
                const long at = (long)(rows.first + here) * A.segments + tid;
                const double sum = A.sum[at];
                s_segment[tid] = s_part[tid][0] = sum == 0.0 ? 0.0 : sum * weight_of(A.most[at], s_most[here], A.c);
            }
            __syncthreads();
            auto segment_of = [&](int d) __attribute__((always_inline)) { return (s_token[s_down[d]] + R.shift) / kPiece / A.pieces; };
            if (tid == 0)
                for (int d = 0; d < down; ++d) {
                    const int g = segment_of(d);
                    const double rest = s_segment[g] - weight_of(s_logit[s_down[d]], s_most[here], A.c);
                    s_segment[g] = rest > 0.0 ? rest : 0.0;
                }
            // what is left of nearly all of a segment may be roundings, with no token behind them: that segment is added up anew
            if (down > 0) {
                __syncthreads();
                uint64_t again = 0;
                for (int d = 0; d < down; ++d) {
                    const int g = segment_of(d);
                    if (s_segment[g] > 0.0 && !(s_segment[g] > kSmall * s_part[g][0])) again |= 1ull << g;
                }
                again = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(again >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)again);
                __syncthreads();  // before measure writes what others may still read
                for (; again != 0; again &= again - 1) measure(__builtin_ctzll(again), __builtin_ctzll(again) + 1);
            }
        }
    }
    __syncthreads();
    // the first segment whose end is past the aim, or the last with anything
    const double mine = lane < A.segments ? s_segment[lane] : 0.0, ends = wave_scan_double(mine, lane);
    const double aim = (double)A.sample[s] * lane_double(ends, kWave - 1);
    const uint64_t passed = ballot(ends > aim && mine > 0.0), any = ballot(mine > 0.0);
    const int segment = passed ? __builtin_ctzll(passed) : any ? 63 - __builtin_clzll(any) : 0;
    double run = segment > 0 ? lane_double(ends, segment - 1) : 0.0;  // the sum before it
    const int end = min((segment + 1) * A.pieces, R.pieces());
    int past = 0x7FFFFFFF, some = -1;  // the first element past the aim, the last with a weight
    for (int p0 = segment * A.pieces; p0 < end; p0 += kWalkThreads) {
        const int p = p0 + tid;
        double w[kPiece], sum = 0.0;
        float x[kPiece];
        R.load(p, end, x);
#pragma unroll
        for (int e = 0; e < kPiece; ++e) {
            w[e] = p < end && !(x[e] == -INFINITY) ? weight(x[e], R.first(p) + e) : 0.0;
            if (w[e] > 0.0) some = (int)(R.first(p) + e);
            sum += w[e];
        }
        double before = wave_scan_double(sum, lane);
        if (lane == kWave - 1) s_scan[wave] = before;
        before -= sum;
        __syncthreads();
        double base = run;
#pragma unroll
        for (int v = 0; v < kWalkWaves; ++v) {
            if (v == wave) before += base;
            base += s_scan[v];
        }
        run = base;
        if (past == 0x7FFFFFFF) {
#pragma unroll
            for (int e = 0; e < kPiece; ++e) {
                before += w[e];
                if (past == 0x7FFFFFFF && w[e] > 0.0 && before > aim) past = (int)(R.first(p) + e);
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int j = 1; j < kWave; j *= 2) {
        past = min(past, __shfl_xor(past, j));
        some = max(some, __shfl_xor(some, j));
    }
    if (lane == 0) {
        s_past[wave] = past;
        s_some[wave] = some;
    }
    __syncthreads();
    if (tid != 0) return;
#pragma unroll
    for (int v = 0; v < kWalkWaves; ++v) {
        past = min(past, s_past[v]);
        some = max(some, s_some[v]);
    }
    A.token[s] = past != 0x7FFFFFFF ? past : some;
}

// The segments' sums of what is left of r behind the first draft turned down, one workgroup each.
template <class T>
__global__ void __launch_bounds__(kStatThreads) verify_rest_kernel(VerifyArgs A) {
    __shared__ float s_most;
    __shared__ double s_sum[kStatThreads / kWave];
    const int s = (int)(blockIdx.x / A.segments), segment = (int)(blockIdx.x - (long)s * A.segments);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const WalkState W = A.state[s];
    if (W.down == 0) return;
    const Rows rows = sequence_rows(A.offsets, s, A.N);
    const Row<T> R(A, rows.first + W.here);
    const float* const q = A.draft + (rows.first + W.down) * A.draft_stride;
    if (wave == 0) {
        const float most = wave_max(lane < A.segments ? A.most[(long)(rows.first + W.here) * A.segments + lane] : -INFINITY);
        if (lane == 0) s_most = most;
    }
    __syncthreads();
    const double scale = 1.0 / W.left;
    const int last = min((segment + 1) * A.pieces, R.pieces());
    double sum = 0.0;
    for (int p0 = segment * A.pieces + tid; p0 < last; p0 += 2 * kStatThreads) {
        typename Row<T>::Raw raw[2];
        float x[2][kPiece], y[2][kPiece];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int p = p0 + k * kStatThreads;
            R.fetch(p, raw[k]);
#pragma unroll
            for (int i = 0; i < kPiece; ++i) y[k][i] = q[min(max(R.first(p) + i, 0L), A.V - 1)];
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            R.values(p0 + k * kStatThreads, last, raw[k], x[k]);
#pragma unroll
            for (int i = 0; i < kPiece; ++i)
                sum += x[k][i] == -INFINITY ? 0.0 : less(weight_of(x[k][i], s_most, A.c), scale, y[k][i]);
        }
    }
    sum = wave_sum_double(sum);
    if (lane == 0) s_sum[wave] = sum;
    __syncthreads();
    if (tid == 0) A.rest[(long)s * A.segments + segment] = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
}

// Elements of a segment: 2048, up to 8192 while there are rows enough, more where a row would have more segments than lanes.  A row's
// first and last piece may hold one element each, so that V elements lie in up to (V + 14) / 8 pieces.
constexpr long kSegment = kStatThreads * kPiece;
long segments_at(long size, long V) { return ((V + 2 * (kPiece - 1)) / kPiece + size / kPiece - 1) / (size / kPiece); }
long segment_of(long N, long V) {
    long size = kSegment;
    while (size < 4 * kSegment && N * (V / (2 * size)) >= 1024) size *= 2;
    while (segments_at(size, V) > kSegments) size *= 2;
    return size;
}
int segments_of(long N, long V) { return (int)segments_at(segment_of(N, V), V); }

template <class T>
int verify(const VerifyArgs& A, int S, bool greedy, hipStream_t stream) {
    const dim3 grid((unsigned)((long)A.N * A.segments));
    const auto stat = greedy ? (A.pieces <= kStatThreads ? verify_stat_kernel<T, true, 1> : A.pieces <= 2 * kStatThreads ? verify_stat_kernel<T, true, 2> : verify_stat_kernel<T, true, 4>)
                             : (A.pieces <= kStatThreads ? verify_stat_kernel<T, false, 1> : A.pieces <= 2 * kStatThreads ? verify_stat_kernel<T, false, 2> : verify_stat_kernel<T, false, 4>);
    hipLaunchKernelGGL(stat, grid, dim3(kStatThreads), 0, stream, A);
    if (reskv_host::check_launch("verify_stat_kernel")) return 1;
    hipLaunchKernelGGL((greedy ? verify_walk_kernel<T, true, false> : verify_walk_kernel<T, false, false>), dim3((unsigned)S), dim3(walk_threads(greedy)), 0,
                       stream, A);
    if (reskv_host::check_launch("verify_walk_kernel")) return 1;
    if (!A.draft) return 0;
    hipLaunchKernelGGL(verify_rest_kernel<T>, dim3((unsigned)((long)S * A.segments)), dim3(kStatThreads), 0, stream, A);
    if (reskv_host::check_launch("verify_rest_kernel")) return 1;
    hipLaunchKernelGGL((verify_walk_kernel<T, false, true>), dim3((unsigned)S), dim3(walk_threads(false)), 0, stream, A);
    return reskv_host::check_launch("verify_walk_kernel");
}

// ---------------------------------------------------------------------------
// accepted tokens moved together
// ---------------------------------------------------------------------------

struct KeepArgs {
    Pool pool;
    long layer;  // bytes of a pool
    const int32_t *starts, *path, *counts;
    int width;
};

// One workgroup per (sequence, KV head, layer), everything through registers: all reads are done before the barrier, all
// writes come behind it, so that a path may be any.  A thread takes (token, quarter): a piece of K's codes, a scaling and a scale
// and lowest value of V; and (group of eight tokens, piece): 16 bytes of V's codes, whose nibbles it gathers token by token.
// Tokens lie in three blocks at most, whose places are looked up once.
//
// Bound: the chain of trips to memory (starts, path and table, codes, codes out) of the workgroups that a CU has in
// turns: 32 trees of 10 to 64 nodes, 32 layers and 8 heads (8192 workgroups) 15 us, one of 8 nodes 4.5.  With 320 threads, one for every item that
// there may be, and a lookup per token it was 32 us.
constexpr int kKeepThreads = 128;  // 64 tokens in two turns, the nine groups of eight that they can lie in in three
__global__ void __launch_bounds__(kKeepThreads) keep_kernel(KeepArgs A) {
    __shared__ int s_from[kNodes];   // source of token starts + j, -1 where nothing moves
    __shared__ char* s_block[4];     // of tokens starts / 32 * 32 on
    const int s = (int)(blockIdx.x / A.pool.heads), h = (int)(blockIdx.x - (long)s * A.pool.heads), tid = threadIdx.x;
    const int start = A.starts[s], count = min(A.counts[s], A.width);
    const bool good = start >= 0 && start <= 0x7FFFFFFF - 2 * kNodes;
    int from = -1;
    if (tid < kNodes) {
        if (tid < count && good) from = A.path[(long)s * A.width + tid];
        if (from < 0 || from >= kNodes || from == tid) from = -1;
        s_from[tid] = from;
    } else if (tid < kNodes + 4 && good) {
        char* const p = A.pool.at(s, start / kBlock + tid - kNodes, h);
        s_block[tid - kNodes] = p ? p + blockIdx.y * A.layer : nullptr;
    }
    if (__syncthreads_or(from >= 0) == 0) return;
    auto block_of = [&](int t) __attribute__((always_inline)) { return s_block[t / kBlock - start / kBlock]; };
    const int part = tid & 3, piece = tid & 31;  // quarter of a token; (c / 64, c % 16)
    const int at = (piece >> 4) * 64 + (piece & 15);
    struct Token {
        char* dst;
        uint4 k;
        uint32_t ks, vs, vl;
    };
    auto read_token = [&](int j) __attribute__((always_inline)) {
        Token x = {};
        const int from = s_from[j], t = start + max(from, 0), in = t & (kBlock - 1);
        char* const src = block_of(t);
        if (from < 0 || !src) return x;
        x.dst = block_of(start + j);
        x.k = reinterpret_cast<const uint4*>(src)[(in >> 4) * 64 + part * 16 + (in & 15)];
        x.ks = reinterpret_cast<const uint32_t*>(src + kKScale)[((in >> 4) * 4 + part) * 16 + (in & 15)];
        x.vs = reinterpret_cast<const uint16_t*>(src + kVScale)[part * kBlock + in];
        x.vl = reinterpret_cast<const uint16_t*>(src + kVLow)[part * kBlock + in];
        return x;
    };
    auto write_token = [&](const Token& x, int j) __attribute__((always_inline)) {
        if (!x.dst) return;
        const int in = (start + j) & (kBlock - 1);
        reinterpret_cast<uint4*>(x.dst)[(in >> 4) * 64 + part * 16 + (in & 15)] = x.k;
        reinterpret_cast<uint32_t*>(x.dst + kKScale)[((in >> 4) * 4 + part) * 16 + (in & 15)] = x.ks;
        reinterpret_cast<uint16_t*>(x.dst + kVScale)[part * kBlock + in] = (uint16_t)x.vs;
        reinterpret_cast<uint16_t*>(x.dst + kVLow)[part * kBlock + in] = (uint16_t)x.vl;
    };
    struct Codes {
        uint4* dst;
        uint4 v;
    };
    auto read_codes = [&](int octet) __attribute__((always_inline)) {
        Codes x = {};
        if (8 * octet >= start + min(count, kNodes)) return x;
        char* const block = block_of(8 * octet);
        if (!block) return x;
        const uint4* src[8];
        uint32_t fresh = 0;  // tokens of the octet that are written
        int nibbles = 0;     // where their nibbles come from, four bits each
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int to = 8 * octet + e - start;
            const int t = to >= 0 && to < kNodes ? s_from[to & (kNodes - 1)] : -1;
            const char* const p = t >= 0 ? block_of(start + max(t, 0)) : nullptr;
            src[e] = reinterpret_cast<const uint4*>((p ? p : block) + kVCodes) + (((start + max(t, 0)) >> 3 & 3) * 16 + at);
            nibbles |= ((start + t) & 7) << (4 * e);
            fresh |= (uint32_t)(p != nullptr) << e;
        }
        if (fresh == 0) return x;
        x.dst = reinterpret_cast<uint4*>(block + kVCodes) + ((octet & 3) * 16 + at);
        x.v = *x.dst;
        // all eight pieces at once; those of tokens that stay are not used
        const uint4 w0 = *src[0], w1 = *src[1], w2 = *src[2], w3 = *src[3], w4 = *src[4], w5 = *src[5], w6 = *src[6], w7 = *src[7];
        auto put = [&](const uint4& w, int e) __attribute__((always_inline)) {
            const int n = nibbles >> (4 * e) & 7, from = 4 * (n / 2 + 4 * (n % 2)), b = nibble(e);
            const uint32_t mask = (fresh >> e & 1 ? 15u : 0u) << b;
            x.v.x = (x.v.x & ~mask) | ((w.x >> from) << b & mask);
            x.v.y = (x.v.y & ~mask) | ((w.y >> from) << b & mask);
            x.v.z = (x.v.z & ~mask) | ((w.z >> from) << b & mask);
            x.v.w = (x.v.w & ~mask) | ((w.w >> from) << b & mask);
        };
        put(w0, 0), put(w1, 1), put(w2, 2), put(w3, 3), put(w4, 4), put(w5, 5), put(w6, 6), put(w7, 7);
        return x;
    };
    constexpr int kStep = kKeepThreads / 32;
    const int octet = (start >> 3) + (tid >> 5), j = tid >> 2;
    const Token t0 = read_token(j), t1 = read_token(j + kKeepThreads / 4);
    const Codes c0 = read_codes(octet), c1 = read_codes(octet + kStep), c2 = read_codes(octet + 2 * kStep);
    __builtin_amdgcn_s_waitcnt(0);  // what was read is here before anybody writes
    __syncthreads();
    write_token(t0, j);
    write_token(t1, j + kKeepThreads / 4);
    if (c0.dst) *c0.dst = c0.v;
    if (c1.dst) *c1.dst = c1.v;
    if (c2.dst) *c2.dst = c2.v;
}

}  // namespace

extern "C" int reskv_draft_tree(const int32_t* parents, const int32_t* offsets, const int32_t* starts, int S, int64_t N, uint64_t* seen,
                                int32_t* positions, void* stream) {
    RESKV_REQUIRE(parents && offsets && seen, "null pointer");
    RESKV_REQUIRE(S > 0 && S < (1 << 25) && N > 0 && N < (1LL << 30), "bad sizes (sequences %d, rows %ld)", S, (long)N);
    hipLaunchKernelGGL(tree_masks_kernel, dim3((unsigned)S), dim3(kWave), 0, (hipStream_t)stream, parents, offsets, starts, (int)N, seen,
                       positions);
    return reskv_host::check_launch("tree_masks_kernel");
}

extern "C" int64_t reskv_verify_workspace_bytes(int S, int64_t N, int64_t V) {
    if (S < 1 || N < 1 || N >= (1LL << 24) || V < 1 || V >= (1LL << 30)) return 0;
    return N * segments_of(N, V) * 16 + S * (segments_of(N, V) * 8LL + (int64_t)sizeof(WalkState));
}

extern "C" int reskv_verify_drafts(const void* logits, int logits_fp32, int64_t row_stride, const int64_t* tokens, const int32_t* parents,
                                   const int32_t* offsets, const float* accept, const float* sample, const float* draft,
                                   int64_t draft_stride, double temperature, int S, int64_t N, int64_t V, int32_t* path, int32_t* counts,
                                   int64_t* token, void* workspace, int64_t workspace_bytes, void* stream) {
    const bool greedy = temperature == 0.0;
    RESKV_REQUIRE(logits && tokens && parents && offsets && path && counts && token && (greedy || (accept && sample)), "null pointer");
    RESKV_REQUIRE(S > 0 && S < (1 << 22) && N > 0 && N < (1LL << 24) && V > 0 && V < (1LL << 30), "bad sizes (sequences %d, rows %ld, tokens %ld)", S,
                  (long)N, (long)V);
    RESKV_REQUIRE(row_stride >= 0 && (!draft || draft_stride >= 0), "row strides must not be negative");
    RESKV_REQUIRE(temperature >= 0.0 && temperature < INFINITY, "temperature must be finite and not negative");
    RESKV_REQUIRE(greedy || temperature >= 1e-30, "a temperature that is not 0 must be 1e-30 or more");
    RESKV_REQUIRE(aligned16(logits) && aligned16(workspace), "logits and the workspace must be 16-byte aligned");
    RESKV_REQUIRE(workspace && workspace_bytes >= reskv_verify_workspace_bytes(S, N, V), "the workspace is too small");
    VerifyArgs A{};
    A.logits = logits;
    A.tokens = tokens;
    A.parents = parents;
    A.offsets = offsets;
    A.accept = accept;
    A.sample = sample;
    A.draft = greedy ? nullptr : draft;
    A.row_stride = row_stride;
    A.draft_stride = draft_stride;
    A.V = V;
    A.path = path;
    A.counts = counts;
    A.token = token;
    A.segments = segments_of(N, V);  // one per lane of the walk
    RESKV_REQUIRE(A.segments <= kSegments, "a row has %d segments, more than %d", A.segments, kSegments);
    A.pieces = (int)(segment_of(N, V) / kPiece);
    A.sum = (double*)workspace;
    A.most = (float*)(A.sum + N * A.segments);
    A.arg = (int32_t*)(A.most + N * A.segments);
    A.rest = (double*)(A.arg + N * A.segments);
    A.state = (WalkState*)(A.rest + (int64_t)S * A.segments);
    A.c = greedy ? 0.0 : 1.4426950408889634074 / temperature;
    A.N = (int)N;
    RESKV_REQUIRE(N * A.segments < kLaunchThreads / kStatThreads && (int64_t)S * A.segments < kLaunchThreads / kStatThreads && S < kLaunchThreads / walk_threads(greedy),
                  "too many rows or sequences");
    return logits_fp32 ? verify<float>(A, S, greedy, (hipStream_t)stream) : verify<uint16_t>(A, S, greedy, (hipStream_t)stream);
}

extern "C" int reskv_int4_keep(void* pages, int layers, int64_t num_pages, int page_tokens, int Hk, const int32_t* table,
                               int table_width, int S, const int32_t* starts, const int32_t* path, int width, const int32_t* counts,
                               void* stream) {
    RESKV_REQUIRE(starts && path && counts, "null pointer");
    if (!pool_ok(pages, num_pages, page_tokens, Hk, table, table_width)) return 1;
    RESKV_REQUIRE(layers > 0 && layers < (1 << 16) && S > 0 && width >= 1 && width <= kNodes, "bad sizes (layers %d, sequences %d, width of a path %d)",
                  layers, S, width);
    RESKV_REQUIRE((long)S * Hk < kLaunchThreads / kKeepThreads, "too many sequences");
    KeepArgs A{};
    A.pool = make_pool(pages, num_pages, page_tokens, Hk, table, table_width);
    A.layer = (long)num_pages * Hk * (page_tokens / kBlock) * kBlockBytes;
    A.starts = starts;
    A.path = path;
    A.counts = counts;
    A.width = width;
    hipLaunchKernelGGL(keep_kernel, dim3((unsigned)(S * Hk), (unsigned)layers), dim3(kKeepThreads), 0, (hipStream_t)stream, A);
    return reskv_host::check_launch("keep_kernel");
}
