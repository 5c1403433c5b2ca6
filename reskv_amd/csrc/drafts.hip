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
constexpr double kSmall = 0x1p-20;    // of a row's sum: what is left of less is added up anew, as a difference has lost its bits
constexpr int kStatThreads = 256, kWalkThreads = 1024, kWalkWaves = kWalkThreads / kWave;

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
    double c;          // log2(e) / temperature
    int N, segments, pieces;  // pieces of a segment
};

// 2^y for y <= 0, to 2^-47 of itself: the series of e^(f ln 2) to the eleventh power for a fraction f of at most a half.  0 below
// 2^-1074; a NaN goes on.
__device__ __forceinline__ double exp2_of(double y) {
    y = y < -1100.0 ? -1100.0 : y;
    const double whole = __builtin_rint(y), z = (y - whole) * 0.69314718055994530942;
    double p = 1.0 / 39916800.0;
    p = __builtin_fma(p, z, 1.0 / 3628800.0);
    p = __builtin_fma(p, z, 1.0 / 362880.0);
    p = __builtin_fma(p, z, 1.0 / 40320.0);
    p = __builtin_fma(p, z, 1.0 / 5040.0);
    p = __builtin_fma(p, z, 1.0 / 720.0);
    p = __builtin_fma(p, z, 1.0 / 120.0);
    p = __builtin_fma(p, z, 1.0 / 24.0);
    p = __builtin_fma(p, z, 1.0 / 6.0);
    p = __builtin_fma(p, z, 0.5);
    p = __builtin_fma(p, z, 1.0);
    p = __builtin_fma(p, z, 1.0);
    return __builtin_ldexp(p, (int)whole);
}

template <class T>
__device__ __forceinline__ float element(const T* p) { return *p; }
template <>
__device__ __forceinline__ float element<uint16_t>(const uint16_t* p) { return h2f(*p); }

// Elements 8 p - shift .. + 7 of a row, whose pieces are 16 bytes of aligned fp16 memory (or twice that of fp32); minus infinity for
// those that are not in the row.
template <class T>
struct Row {
    const T* p;
    int shift;
    __device__ __forceinline__ Row(const VerifyArgs& A, int row)
        : p((const T*)A.logits + row * A.row_stride), shift((int)(((uintptr_t)p & 15) / sizeof(T))) {}
    __device__ __forceinline__ long first(int piece) const { return (long)piece * kPiece - shift; }
    __device__ __forceinline__ void load(const VerifyArgs& A, int piece, float* x) const {
        const long at = first(piece);
        if (at >= 0 && at + kPiece <= A.V) {
            uint4 w[sizeof(T) / 2];
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const uint4*>(p + at)[i];
            const uint32_t d[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
            if (sizeof(T) == 2) {
#pragma unroll
                for (int i = 0; i < kPiece; ++i) x[i] = h2f((uint16_t)(d[i >> 1] >> (16 * (i & 1))));
            } else {
                const uint4 v = w[sizeof(T) / 2 - 1];
                const uint32_t e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int i = 0; i < kPiece; ++i) x[i] = i2f((int)(i < 4 ? d[i & 3] : e[i & 3]));
            }
        } else {
#pragma unroll
            for (int i = 0; i < kPiece; ++i) x[i] = at + i >= 0 && at + i < A.V ? element(p + at + i) : -INFINITY;
        }
    }
};

__device__ __forceinline__ double wave_sum_double(double v) {
#pragma unroll
    for (int i = 1; i < kWave; i *= 2) v += __shfl_xor(v, i);
    return v;
}

// Each row's segments: the largest logit and the sum of exp2((x - largest) c) in 64 bits, or where the largest is.  A thread
// keeps its own maximum and brings its sum down when that moves.
template <class T, bool GREEDY>
__global__ void __launch_bounds__(kStatThreads) verify_stat_kernel(VerifyArgs A) {
    __shared__ float s_most[kStatThreads / kWave];
    __shared__ double s_sum[kStatThreads / kWave];
    __shared__ int s_arg[kStatThreads / kWave];
    const int row = (int)(blockIdx.x / A.segments), segment = (int)(blockIdx.x - (long)row * A.segments);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const Row<T> R(A, row);
    const int last = (int)min((long)(segment + 1) * A.pieces, (A.V + R.shift + kPiece - 1) / kPiece);
    float most = -INFINITY;
    double sum = 0.0;
    int arg = 0x7FFFFFFF;
    bool nan = false;
    for (int p = segment * A.pieces + tid; p < last; p += kStatThreads) {
        float x[kPiece];
        R.load(A, p, x);
        if (GREEDY) {
#pragma unroll
            for (int i = 0; i < kPiece; ++i) {
                const long at = R.first(p) + i;
                nan |= x[i] != x[i];
                if (at >= 0 && at < A.V && (x[i] > most || arg == 0x7FFFFFFF)) {
                    most = x[i];
                    arg = (int)at;
                }
            }
        } else {
            float top = x[0];
#pragma unroll
            for (int i = 1; i < kPiece; ++i) top = fmaxf(top, x[i]);
            if (top > most) {
                sum *= exp2_of(((double)most - (double)top) * A.c);  // nothing yet: 0 times 0
                most = top;
            }
#pragma unroll
            for (int i = 0; i < kPiece; ++i)
                if (!(x[i] == -INFINITY)) sum += exp2_of(((double)x[i] - (double)most) * A.c);
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
        sum = most == wave_most || sum == 0.0 ? sum : sum * exp2_of(((double)most - (double)wave_most) * A.c);
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
            all += s_most[w] == top || s_sum[w] == 0.0 ? s_sum[w] : s_sum[w] * exp2_of(((double)s_most[w] - (double)top) * A.c);
        A.sum[at] = all;
    }
}

// The walk down a tree, one workgroup per sequence.  Everything that the decisions need comes in one trip to memory, a lane
// per node: the node's token, its logit behind its parent, its draft probability, and its row's statistics from the
// segments.  After that only a draft that was turned down costs a pass over a row (with `draft`: the sums of what is left), and the
// token at the end one over a segment.
template <class T, bool GREEDY>
__global__ void __launch_bounds__(kWalkThreads) verify_walk_kernel(VerifyArgs A) {
    __shared__ double s_total[kNodes];  // of a node's row: sum of exp2((x - most) c)
    __shared__ float s_most[kNodes], s_logit[kNodes], s_q[kNodes], s_accept[kNodes];
    __shared__ int s_parent[kNodes], s_token[kNodes], s_best[kNodes], s_path[kNodes];
    __shared__ double s_segment[kSegments];        // what is left of r, by segment
    __shared__ double s_scan[kWalkWaves];
    __shared__ int s_down[kNodes];                 // drafts turned down at the node reached: their nodes,
    __shared__ double s_scale[kNodes];             // and one over the sum of r before them
    const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Rows rows = sequence_rows(A.offsets, s, A.N);
    const int n = min(rows.count, kNodes);
    if (n == 0) {
        if (tid < kNodes) A.path[(long)s * kNodes + tid] = -1;
        if (tid == 0) {
            A.counts[s] = 0;
            A.token[s] = -1;
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
    }
    for (int i = wave; i < n; i += kWalkWaves) {
        const long at = (long)(rows.first + i) * A.segments + lane;
        const bool in = lane < A.segments;
        const float most = in ? A.most[at] : -INFINITY, top = wave_max(most);
        if (GREEDY) {
            const int arg = in ? A.arg[at] : 0x7FFFFFFF;
            int best = most == top || arg == -1 ? arg : 0x7FFFFFFF;
#pragma unroll
            for (int j = 1; j < kWave; j *= 2) best = min(best, __shfl_xor(best, j));
            if (lane == 0) s_best[i] = best;
        } else {
            double sum = in ? A.sum[at] : 0.0;
            if (sum != 0.0 && most != top) sum *= exp2_of(((double)most - (double)top) * A.c);
            sum = wave_sum_double(sum);
            if (lane == 0) {
                s_total[i] = sum;
                s_most[i] = top;
            }
        }
    }
    __syncthreads();

    int here = 0, length = 1;
    if (tid == 0) s_path[0] = 0;
    if (GREEDY) {
        for (int i = 1; i < n; ++i)
            if (s_parent[i] == here && s_token[i] == s_best[here]) {
                here = i;
                if (tid == 0) s_path[length] = i;
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
        double w = x == -INFINITY ? 0.0 : exp2_of(((double)x - (double)s_most[here]) * A.c);
        for (int i = 0; i < down; ++i) {
            if (A.draft) {
                const double rest = w * s_scale[i] - (double)A.draft[(rows.first + s_down[i]) * A.draft_stride + at];
                w = rest > 0.0 ? rest : 0.0;
            } else if (s_token[s_down[i]] == at) {
                w = 0.0;
            }
        }
        return w;
    };
    const int64_t pieces_all = A.pieces;
    // The segments' sums of r, by whole waves; returns their sum.
    auto measure = [&]() __attribute__((always_inline)) {
        const Row<T> R(A, rows.first + here);
        for (int g = wave; g < A.segments; g += kWalkWaves) {
            const int last = (int)min((g + 1) * pieces_all, (A.V + R.shift + kPiece - 1) / kPiece);
            double sum = 0.0;
            for (int p = g * A.pieces + lane; p < last; p += kWave) {
                float x[kPiece];
                R.load(A, p, x);
#pragma unroll
                for (int i = 0; i < kPiece; ++i)
                    if (!(x[i] == -INFINITY)) sum += weight(x[i], R.first(p) + i);
            }
            sum = wave_sum_double(sum);
            if (lane == 0) s_segment[g] = sum;
        }
        __syncthreads();
        double all = 0.0;
        for (int g = 0; g < A.segments; ++g) all += s_segment[g];
        __syncthreads();
        return all;
    };
    left = s_total[0];
    for (int i = 1; i < n && left > 0.0 && left < INFINITY; ++i) {
        if (s_parent[i] != here) continue;
        const int t = s_token[i];
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
        __syncthreads();
        if (tid == 0) {
            s_down[down] = i;
            s_scale[down] = 1.0 / left;
        }
        __syncthreads();
        ++down;
        // without a distribution only one token goes; where that is nearly all, the rest is added up anew
        double rest = left - w;
        if (A.draft || !(rest > kSmall * s_total[here])) {
            rest = measure();
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
    if (tid == 0) A.counts[s] = length;
    if (!(left > 0.0 && left < INFINITY)) {
        if (tid == 0) A.token[s] = -1;
        return;
    }
    const Row<T> R(A, rows.first + here);
    if (whole) {
        if ((A.draft && down > 0) || !(left > kSmall * s_total[here])) {
            measure();
        } else {
            // from the row's statistics, without the tokens turned down
            if (tid < A.segments) {
                const long at = (long)(rows.first + here) * A.segments + tid;
                const double sum = A.sum[at];
                s_segment[tid] = sum == 0.0 ? 0.0 : sum * exp2_of(((double)A.most[at] - (double)s_most[here]) * A.c);
            }
            __syncthreads();
            if (tid == 0)
                for (int i = 0; i < down; ++i) {
                    const int g = (s_token[s_down[i]] + R.shift) / kPiece / A.pieces;
                    const double rest = s_segment[g] - exp2_of(((double)s_logit[s_down[i]] - (double)s_most[here]) * A.c);
                    s_segment[g] = rest > 0.0 ? rest : 0.0;
                }
        }
    }
    __syncthreads();
    double all = 0.0;
    for (int g = 0; g < A.segments; ++g) all += s_segment[g];
    const double aim = (double)A.sample[s] * all;
    int segment = 0;
    double run = 0.0;
    for (int g = 0; g < A.segments; ++g) {  // the first that passes the aim, or the last with anything
        const double mine = s_segment[g];
        if (mine > 0.0) segment = g;
        if (run + mine > aim) break;
        if (g + 1 < A.segments) run += mine;
    }
    // (run: the sum before `segment`, where the aim was passed there)
    run = 0.0;
    for (int g = 0; g < segment; ++g) run += s_segment[g];
    const int end = (int)min((segment + 1) * pieces_all, (A.V + R.shift + kPiece - 1) / kPiece);
    int past = 0x7FFFFFFF, some = -1;  // the first element past the aim, the last with a weight
    for (int p0 = segment * A.pieces; p0 < end; p0 += kWalkThreads) {
        const int p = p0 + tid;
        double w[kPiece], sum = 0.0;
        float x[kPiece];
        if (p < end) R.load(A, p, x);
#pragma unroll
        for (int i = 0; i < kPiece; ++i) {
            w[i] = p < end && !(x[i] == -INFINITY) ? weight(x[i], R.first(p) + i) : 0.0;
            if (w[i] > 0.0) some = (int)(R.first(p) + i);
            sum += w[i];
        }
        double before = sum;  // inclusive sums over the lanes
#pragma unroll
        for (int i = 1; i < kWave; i *= 2) {
            const double other = __shfl_up(before, i);
            if (lane >= i) before += other;
        }
        if (lane == kWave - 1) s_scan[wave] = before;
        before -= sum;
        __syncthreads();
        double base = run;
        for (int v = 0; v < kWalkWaves; ++v) {
            if (v == wave) before += base;
            base += s_scan[v];
        }
        run = base;
        if (past == 0x7FFFFFFF) {
#pragma unroll
            for (int i = 0; i < kPiece; ++i) {
                before += w[i];
                if (past == 0x7FFFFFFF && w[i] > 0.0 && before > aim) past = (int)(R.first(p) + i);
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 1; i < kWave; i *= 2) {
        past = min(past, __shfl_xor(past, i));
        some = max(some, __shfl_xor(some, i));
    }
    __shared__ int s_past[kWalkWaves], s_some[kWalkWaves];
    if (lane == 0) {
        s_past[wave] = past;
        s_some[wave] = some;
    }
    __syncthreads();
    if (tid != 0) return;
    for (int v = 0; v < kWalkWaves; ++v) {
        past = min(past, s_past[v]);
        some = max(some, s_some[v]);
    }
    A.token[s] = past != 0x7FFFFFFF ? past : some;
}

// Segments of a row: 8192 elements each, down to 2048 while the rows are few.
int segments_of(long N, long V) {
    const long most = (V + 2047) / 2048, wide = (V + 8191) / 8192, wanted = (1024 + N - 1) / N;
    const long n = wide > wanted ? wide : wanted < most ? wanted : most;
    return (int)(n < 1 ? 1 : n > kSegments ? kSegments : n);
}

template <class T>
int verify(const VerifyArgs& A, int S, bool greedy, hipStream_t stream) {
    const dim3 grid((unsigned)((long)A.N * A.segments));
    hipLaunchKernelGGL((greedy ? verify_stat_kernel<T, true> : verify_stat_kernel<T, false>), grid, dim3(kStatThreads), 0, stream, A);
    if (reskv_host::check_launch("verify_stat_kernel")) return 1;
    hipLaunchKernelGGL((greedy ? verify_walk_kernel<T, true> : verify_walk_kernel<T, false>), dim3((unsigned)S), dim3(kWalkThreads), 0, stream, A);
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
// writes come behind it, so that a path may be any.  Threads 0 .. 255 take (token, quarter): a piece of K's codes, a
// scaling and a scale and lowest value of V; all 320 take the 16-byte pieces of V's codes that get tokens, (group of eight
// tokens, piece), and gather their nibbles token by token.
constexpr int kKeepThreads = 320;
__global__ void __launch_bounds__(kKeepThreads) keep_kernel(KeepArgs A) {
    __shared__ int s_from[kNodes];  // source of token starts + j, -1 where nothing moves
    const int s = (int)(blockIdx.x / A.pool.heads), h = (int)(blockIdx.x - (long)s * A.pool.heads), tid = threadIdx.x;
    const int start = A.starts[s], count = min(A.counts[s], A.width);
    int from = -1;
    if (tid < kNodes) {
        if (tid < count) from = A.path[(long)s * A.width + tid];
        if (from < 0 || from >= kNodes || from == tid || start < 0 || start > 0x7FFFFFFF - 2 * kNodes) from = -1;
        s_from[tid] = from;
    }
    if (__syncthreads_or(from >= 0) == 0) return;
    char* const base = A.pool.pages + blockIdx.y * A.layer;
    // block of a token in this layer; null without a page
    auto block_of = [&](int t) __attribute__((always_inline)) {
        char* const p = A.pool.at(s, t / kBlock, h);
        return p ? base + (p - A.pool.pages) : nullptr;
    };
    uint4 k = {}, v = {};
    uint32_t ks = 0, vs = 0, vl = 0, fresh = 0;
    char *dst = nullptr, *v_dst = nullptr;
    const int j = tid >> 2, part = tid & 3;
    const int t_dst = start + j, in_dst = t_dst & (kBlock - 1);
    if (tid < 4 * kNodes && s_from[j] >= 0) {
        const int t = start + s_from[j], in = t & (kBlock - 1);
        const char* const src = block_of(t);
        dst = block_of(t_dst);
        if (src && dst) {
            k = reinterpret_cast<const uint4*>(src)[(in >> 4) * 64 + part * 16 + (in & 15)];
            ks = reinterpret_cast<const uint32_t*>(src + kKScale)[((in >> 4) * 4 + part) * 16 + (in & 15)];
            vs = reinterpret_cast<const uint16_t*>(src + kVScale)[part * kBlock + in];
            vl = reinterpret_cast<const uint16_t*>(src + kVLow)[part * kBlock + in];
        } else {
            dst = nullptr;
        }
    }
    const int octet = (start >> 3) + (tid >> 5), piece = tid & 31;  // eight tokens; (c / 64, c % 16)
    const int in8 = (octet & 3) * 16 + (piece >> 4) * 64 + (piece & 15);
    if (8 * octet < start + kNodes) {
        for (int e = 0; e < 8; ++e) {
            const int to = 8 * octet + e - start;
            if (to < 0 || to >= kNodes || s_from[to] < 0) continue;
            const int t = start + s_from[to], in = t & (kBlock - 1);
            const char* const src = block_of(t);
            if (!v_dst) v_dst = block_of(8 * octet);
            if (!src || !v_dst) continue;
            if (fresh == 0) v = reinterpret_cast<const uint4*>(v_dst + kVCodes)[in8];
            const uint4 w = reinterpret_cast<const uint4*>(src + kVCodes)[(in >> 3) * 16 + (piece >> 4) * 64 + (piece & 15)];
            const int a = nibble(in & 7), b = nibble(e);
            const uint32_t keep = ~(15u << b);
            v.x = (v.x & keep) | ((w.x >> a) & 15u) << b;
            v.y = (v.y & keep) | ((w.y >> a) & 15u) << b;
            v.z = (v.z & keep) | ((w.z >> a) & 15u) << b;
            v.w = (v.w & keep) | ((w.w >> a) & 15u) << b;
            fresh = 1;
        }
    }
    __builtin_amdgcn_s_waitcnt(0);  // what was read is here before anybody writes
    __syncthreads();
    if (dst) {
        reinterpret_cast<uint4*>(dst)[(in_dst >> 4) * 64 + part * 16 + (in_dst & 15)] = k;
        reinterpret_cast<uint32_t*>(dst + kKScale)[((in_dst >> 4) * 4 + part) * 16 + (in_dst & 15)] = ks;
        reinterpret_cast<uint16_t*>(dst + kVScale)[part * kBlock + in_dst] = (uint16_t)vs;
        reinterpret_cast<uint16_t*>(dst + kVLow)[part * kBlock + in_dst] = (uint16_t)vl;
    }
    if (fresh) reinterpret_cast<uint4*>(v_dst + kVCodes)[in8] = v;
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
    return N * segments_of(N, V) * 16;
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
    A.segments = segments_of(N, V);
    A.pieces = (int)((V / kPiece + 2 + A.segments - 1) / A.segments);
    A.sum = (double*)workspace;
    A.most = (float*)(A.sum + N * A.segments);
    A.arg = (int32_t*)(A.most + N * A.segments);
    A.c = greedy ? 0.0 : 1.4426950408889634074 / temperature;
    A.N = (int)N;
    RESKV_REQUIRE(N * A.segments < kLaunchThreads / kStatThreads, "too many rows");
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
