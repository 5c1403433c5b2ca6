// Paged cache of 4-bit keys and values: rows into pages, rows back, the attention of single
// tokens that reads the pages, and page copies.  include/reskv_serving.h has the layout.
//
// The layout is that of the matrix cores' operands: a lane's 16-byte piece of a block holds
// the codes that it multiplies, eight along the inner dimension per dword (eight channels
// of a token for K, eight tokens of a channel for V), so that the attention takes them from
// memory to v_mfma_f32_16x16x32_f16 without the LDS.  A code becomes an fp16 number by
// masking alone: the bits 0 .. 15 of a nibble at bit 0 are the denormal code * 2^-24, at
// bit 4 the number code * 2^-20 (the matrix cores keep denormals); the other operand carries
// the factor 16 and the result the factor 2^24, both exact.
#include "int4.h"
#include "reskv_drafts.h"

using namespace reskv;

namespace {

// ---------------------------------------------------------------------------
// rows into pages and back
// ---------------------------------------------------------------------------

// Range of a group of 32 channels, of which this lane has 16 and the lane next to it the others.
// `maximum` and `minimum` hand a NaN on.
struct Group {
    float low, scale;
    uint16_t low16, scale16;
};
__device__ __forceinline__ Group group_of(const half2_t* x) {
    half2_t lo = x[0], hi = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
        lo = __builtin_elementwise_minimum(lo, x[i]);
        hi = __builtin_elementwise_maximum(hi, x[i]);
    }
    lo = __builtin_elementwise_minimum(lo, __builtin_bit_cast(half2_t, dpp_u<0xB1>(__builtin_bit_cast(uint32_t, lo))));
    hi = __builtin_elementwise_maximum(hi, __builtin_bit_cast(half2_t, dpp_u<0xB1>(__builtin_bit_cast(uint32_t, hi))));
    const float low = (float)__builtin_elementwise_minimum(lo[0], lo[1]);
    const float high = (float)__builtin_elementwise_maximum(hi[0], hi[1]);
    if (!(high < INFINITY && low > -INFINITY)) return {0.0f, 0.0f, 0x7E00, 0x7E00};
    const float range = high - low;
    float scale = range / 15.0f;
    // a range of more than 24 bits: 64 bits hold it
    if (high - range != low || low + range != high) scale = (float)(((double)high - (double)low) / 15.0);
    const uint16_t scale16 = f2h(scale);
    return {low, h2f(scale16), f2h(low), scale16};
}

// The codes of 16 values: exactly rint((x - low) / scale), at most 15.  The product with the
// reciprocal is within 2^-17 of the quotient (four roundings of 2^-23 at most, of a number below 2^5;
// larger ones become 15); where it is nearer than 2^-16 to a half, 64 bits decide, which hold both sides
// exactly.  That is one value in 2^15.
__device__ __forceinline__ void codes_of(const half2_t* x, const Group& g, uint32_t* code) {
    const float inv = g.scale > 0.0f ? __builtin_amdgcn_rcpf(g.scale) : 0.0f;
    bool near_half = false;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float q = ((float)x[i >> 1][i & 1] - g.low) * inv;
        near_half |= fabsf(__builtin_amdgcn_fractf(q) - 0.5f) < 0x1p-16f;
        code[i] = (uint32_t)fminf(rintf(q), 15.0f);
    }
    if (!near_half) return;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float v = (float)x[i >> 1][i & 1], q = (v - g.low) * inv;
        if (q < 16.0f && fabsf(__builtin_amdgcn_fractf(q) - 0.5f) < 0x1p-16f) {
            const float below = floorf(q), half_way = below + 0.5f;
            const double side = ((double)v - (double)g.low) - (double)half_way * (double)g.scale;
            const float r = side < 0.0 ? below : side > 0.0 ? below + 1.0f : 2.0f * rintf(0.5f * half_way);
            code[i] = (uint32_t)fminf(r, 15.0f);
        }
    }
}

// Rotation of K and Q to their positions on the way into the pages.
struct Turn {
    const uint16_t* q;         // [N, heads * G, 128], null: K and V alone
    uint16_t* q_out;           // [N, heads * G, 128]
    const int32_t* positions;  // per row; null: the token's place in its sequence
    const float *cos, *sin;    // [rows, half]
    long q_token, q_head;      // strides of q in halves
    int G, rows, half, interleaved;
};

// Channels [at, at + 8) of a head whose rotated channels come in pairs: (i, i + half), or (2 i, 2 i + 1) when
// interleaved.  Products and sums are rounded to fp32 one by one and the result to fp16, as the torch formula does it
// and reskv_llama_qkv_rope: pages hold the same bits whichever way a token came.
__device__ __forceinline__ uint4 turned_piece(const Turn& R, const uint16_t* head, int at, int position) {
#pragma clang fp contract(off)
    const uint4 x = *reinterpret_cast<const uint4*>(head + at);
    if (at >= 2 * R.half) return x;
    const uint32_t xw[4] = {x.x, x.y, x.z, x.w};
    uint32_t out[4];
    const long table = (long)position * R.half;
    auto times = [](uint32_t w, int upper) { return h2f((uint16_t)(upper ? w >> 16 : w)); };
    if (R.interleaved) {
        const float4 c = *reinterpret_cast<const float4*>(R.cos + table + at / 2), s = *reinterpret_cast<const float4*>(R.sin + table + at / 2);
        const float cs[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = times(xw[i], 0), b = times(xw[i], 1);
            out[i] = pack_halves(a * cs[i] - b * sn[i], b * cs[i] + a * sn[i]);
        }
    } else {
        const bool second = at >= R.half;
        const int i0 = second ? at - R.half : at;
        const uint4 y = *reinterpret_cast<const uint4*>(head + (second ? i0 : at + R.half));
        const uint32_t yw[4] = {y.x, y.y, y.z, y.w};
        const float4* const c = reinterpret_cast<const float4*>(R.cos + table + i0);
        const float4* const s = reinterpret_cast<const float4*>(R.sin + table + i0);
        const float4 c0 = c[0], c1 = c[1], s0 = s[0], s1 = s[1];
        const float cs[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w}, sn[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float r[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float mine = times(xw[i], e) * cs[2 * i + e], other = times(yw[i], e) * sn[2 * i + e];
                r[e] = second ? mine + other : mine - other;
            }
            out[i] = pack_halves(r[0], r[1]);
        }
    }
    return make_uint4(out[0], out[1], out[2], out[3]);
}

// Rows' queries of KV head h: eight threads per (row, query head), 16 channels each; a workgroup takes kQueries of a block's
// (row, query head), two to a thread.
constexpr int kQueries = 2 * kThreads / 8;
__device__ __forceinline__ void turn_queries(const RowArgs& A, const Turn& R, const Part& P, int h, int set) {
    const int at = 16 * ((int)threadIdx.x & 7), all = (P.hi - P.lo) * R.G;
    uint4 x[2][2];
    uint4* dst[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int u = set * kQueries + i * (kThreads / 8) + ((int)threadIdx.x >> 3);
        dst[i] = nullptr;
        if (u >= all) continue;
        const int t = u / R.G, head = h * R.G + u - t * R.G;
        const long row = P.row + t;
        const int position = R.positions ? R.positions[row] : P.block * kBlock + P.lo + t;
        const bool in = position >= 0 && position < R.rows;
        if (!in && !A.clear_rest) continue;
        dst[i] = reinterpret_cast<uint4*>(R.q_out + (row * A.pool.heads * R.G + head) * kDim + at);
        x[i][0] = x[i][1] = make_uint4(0, 0, 0, 0);
        if (!in) continue;
        const uint16_t* const src = R.q + row * R.q_token + head * R.q_head;
        x[i][0] = turned_piece(R, src, at, position);
        x[i][1] = turned_piece(R, src, at + 8, position);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (!dst[i]) continue;
        dst[i][0] = x[i][0];
        dst[i][1] = x[i][1];
    }
}

// Queries of no sequence get zeros from the workgroups behind the last item (there is always one).
__device__ void clear_queries(const RowArgs& A, const Turn& R, int spare, int spares, int h) {
    const int begin = min(max(A.offsets[0], 0), A.N), end = min(max(A.offsets[A.sequences], begin), A.N);
    const long pieces = (long)R.G * (kDim / 8), rest = (begin + A.N - end) * pieces;
    for (long i = (long)spare * kThreads + threadIdx.x; i < rest; i += (long)spares * kThreads) {
        const long r = i / pieces, row = r < begin ? r : end + r - begin;
        reinterpret_cast<uint4*>(R.q_out + (row * A.pool.heads + h) * R.G * kDim)[i - r * pieces] = make_uint4(0, 0, 0, 0);
    }
}

// One workgroup per (block of 32 tokens that gets rows, head); thread (token, part) has 16 channels
// of K and of V, so that a wave has the eight tokens that share the dwords of V.  With TURN, K is rotated before it is
// quantised, the KV head's queries are rotated beside it, and a row whose position lies outside the tables is left out.
//
// Bound: memory (512 bytes in and 160 out per token and head), with the vector ALU close behind: 37,200 tokens of 8 heads
// in 47 us (4.2 TB/s; a large copy reaches 4.8).  With a division per code and V transposed byte by byte through the
// LDS it was 74 us.  32 single tokens: 6 us, a chain of five trips to memory (offsets, page, rows, old nibbles, out).
// With TURN, 49,100 tokens of 32 / 8 heads (22 KB in and out each) 265 to 277 us, 4 TB/s; 667 nodes of 32 trees 10 us, where it was 15
// with a workgroup's queries before its keys.
template <bool TURN>
__global__ void __launch_bounds__(kThreads) append_kernel(RowArgs A, Turn R) {
    __shared__ __align__(16) uint32_t s_k[512], s_v[512];  // codes as stored
    __shared__ uint32_t s_kp[128];                         // K scalings as stored
    __shared__ uint16_t s_vp[256];                         // V scales and lowest values as stored
    __shared__ bool s_in[kBlock];                          // TURN: tokens whose position is in the tables
    const int h = (int)blockIdx.x % A.pool.heads, item = (int)blockIdx.x / A.pool.heads;
    const Part P = row_part(A, item);
    if (P.seq < 0) {
        if (TURN && blockIdx.y == 0 && A.clear_rest && R.q && A.offsets && P.block >= 0 && P.hi == 0) {
            const int first = item - P.block;  // the number of items
            clear_queries(A, R, P.block, (int)gridDim.x / A.pool.heads - first, h);
        }
        return;
    }
    if (TURN && blockIdx.y > 0) {
        turn_queries(A, R, P, h, (int)blockIdx.y - 1);
        return;
    }
    const int tid = threadIdx.x, token = tid >> 3, part = tid & 7, group = part >> 1;
    bool mine = token >= P.lo && token < P.hi;
    uint4 kw[2] = {}, vw[2] = {};
    if (mine) {
        const long row = P.row + token - P.lo;
        const uint16_t* const key = A.k + row * A.k_token + h * A.k_head;
        const uint4* ks = reinterpret_cast<const uint4*>(key) + 2 * part;
        const uint4* vs = reinterpret_cast<const uint4*>(A.v + row * A.v_token + h * A.v_head) + 2 * part;
        vw[0] = vs[0], vw[1] = vs[1];
        if (TURN) {
            const int position = R.positions ? R.positions[row] : P.block * kBlock + token;
            mine = position >= 0 && position < R.rows;
            if (mine) {
                kw[0] = turned_piece(R, key, 16 * part, position);
                kw[1] = turned_piece(R, key, 16 * part + 8, position);
            }
        } else {
            kw[0] = ks[0], kw[1] = ks[1];
        }
    }
    if (TURN && part == 0) s_in[token] = mine;
    // whether token t of the block is stored (TURN: behind the barrier)
    auto stored = [&](int t) { return t >= P.lo && t < P.hi && (!TURN || s_in[t]); };
    char* const block = A.pool.at(P.seq, P.block, h);
    if (!block) return;
    uint32_t code[16];
    half2_t x[8];
    auto unpack = [&](const uint4* w) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            x[4 * i] = __builtin_bit_cast(half2_t, w[i].x);
            x[4 * i + 1] = __builtin_bit_cast(half2_t, w[i].y);
            x[4 * i + 2] = __builtin_bit_cast(half2_t, w[i].z);
            x[4 * i + 3] = __builtin_bit_cast(half2_t, w[i].w);
        }
    };
    {
        unpack(kw);
        const Group g = group_of(x);
        codes_of(x, g, code);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            uint32_t packed = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) packed |= code[8 * q + e] << nibble(e);
            s_k[(((token >> 4) * 4 + 2 * (part & 1) + q) * 16 + (token & 15)) * 4 + group] = packed;
        }
        if ((part & 1) == 0) s_kp[((token >> 4) * 4 + group) * 16 + (token & 15)] = g.scale16 | ((uint32_t)g.low16 << 16);
    }
    {
        unpack(vw);
        const Group g = group_of(x);
        codes_of(x, g, code);
        if ((part & 1) == 0) {
            s_vp[group * kBlock + token] = g.scale16;
            s_vp[128 + group * kBlock + token] = g.low16;
        }
        // the eight tokens' nibbles of a channel come together over the lanes (token, part) of the wave: each
        // of three exchanges halves the channels that a lane still has, and joins two tokens' nibbles
        const int e = token & 7, shift = 4 * (e / 2 + 4 * (e % 2));
#pragma unroll
        for (int i = 0; i < 16; ++i) code[i] <<= shift;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const auto r = __builtin_amdgcn_permlane32_swap(code[i], code[i + 8], false, false);
            code[i] = r[0] | r[1];  // channels i of lanes below 32, i + 8 of the others
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const auto r = __builtin_amdgcn_permlane16_swap(code[i], code[i + 4], false, false);
            code[i] = r[0] | r[1];
        }
        const bool upper = (token & 1) != 0;  // lane ^ 8 is the token next to it
        const uint32_t keep0 = upper ? code[2] : code[0], keep1 = upper ? code[3] : code[1];
        const uint32_t give0 = upper ? code[0] : code[2], give1 = upper ? code[1] : code[3];
        const int n = 8 * ((token >> 2) & 1) + 4 * ((token >> 1) & 1) + 2 * (token & 1);  // channel in the part
        const int at = (part >> 2) * 256 + ((token >> 3) * 16 + n) * 4 + (part & 3);
        s_v[at] = keep0 | dpp_u<0x128>(give0);  // row_ror:8
        s_v[at + 4] = keep1 | dpp_u<0x128>(give1);
    }
    __syncthreads();
    if (tid < 128) {
        const int t = (tid >> 6) * 16 + (tid & 15);  // the token of both: piece (tile, quarter, token), dword (tile, group, token)
        if (stored(t)) {
            reinterpret_cast<uint4*>(block)[tid] = reinterpret_cast<const uint4*>(s_k)[tid];
            reinterpret_cast<uint32_t*>(block + kKScale)[tid] = s_kp[tid];
        }
    }
    if (stored(tid & 31))  // half (scale or low, group, token)
        reinterpret_cast<uint16_t*>(block + kVScale)[tid] = s_vp[tid];
    // V codes: dword (c / 64, t / 8, c % 16, c / 16 % 4) has the eight tokens of a channel; of a dword whose
    // tokens are not all new the others' nibbles stay
    if (tid < 128) {
        const int t0 = 8 * ((tid >> 4) & 3);
        uint32_t fresh = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (stored(t0 + i)) fresh |= 15u << nibble(i);
        if (fresh == 0) return;
        uint4* const dst = reinterpret_cast<uint4*>(block + kVCodes) + tid;
        uint4 w = reinterpret_cast<const uint4*>(s_v)[tid];
        if (fresh != ~0u) {
            const uint4 old = *dst;
            w.x = (w.x & fresh) | (old.x & ~fresh);
            w.y = (w.y & fresh) | (old.y & ~fresh);
            w.z = (w.z & fresh) | (old.z & ~fresh);
            w.w = (w.w & fresh) | (old.w & ~fresh);
        }
        *dst = w;
    }
}

// Rows of no sequence get zeros from the workgroups behind the last item (there is always one).
__device__ void clear_rows(const RowArgs& A, int spare, int spares, int h) {
    const int begin = min(max(A.offsets[0], 0), A.N);
    const int end = A.sequences > 0 ? min(max(A.offsets[A.sequences], begin), A.N) : begin;
    const int tid = threadIdx.x, rest = begin + A.N - end;
    for (int i = spare * 16 + tid / 16; i < rest; i += spares * 16) {
        const long row = ((long)(i < begin ? i : end + i - begin) * A.pool.heads + h) * kDim;
        reinterpret_cast<uint4*>(A.k_out + row)[tid % 16] = make_uint4(0, 0, 0, 0);
        reinterpret_cast<uint4*>(A.v_out + row)[tid % 16] = make_uint4(0, 0, 0, 0);
    }
}

// The same workgroups the other way.  Bound: memory, 37,200 tokens of 8 heads in 34 us (5.9 TB/s).
__global__ void __launch_bounds__(kThreads) gather_kernel(RowArgs A) {
    __shared__ __align__(16) uint32_t s_v[512];
    __shared__ uint32_t s_vp[128];
    const int h = (int)blockIdx.x % A.pool.heads, items = (int)gridDim.x / A.pool.heads;
    const int item = (int)blockIdx.x / A.pool.heads;
    const Part P = row_part(A, item);
    if (P.seq < 0) {
        if (A.clear_rest && A.offsets && P.block >= 0 && P.hi == 0) {
            const int first = item - P.block;  // the number of items
            clear_rows(A, P.block, items - first, h);
        }
        return;
    }
    const char* const block = A.pool.at(P.seq, P.block, h);
    const int tid = threadIdx.x, token = tid >> 3, part = tid & 7, group = part >> 1;
    const bool mine = token >= P.lo && token < P.hi;
    const long row = ((P.row + token - P.lo) * A.pool.heads + h) * kDim + 16 * part;
    if (!block) {
        if (A.clear_rest && mine)
            for (int i = 0; i < 2; ++i) {
                reinterpret_cast<uint4*>(A.k_out + row)[i] = make_uint4(0, 0, 0, 0);
                reinterpret_cast<uint4*>(A.v_out + row)[i] = make_uint4(0, 0, 0, 0);
            }
        return;
    }
    if (tid < 128) {
        reinterpret_cast<uint4*>(s_v)[tid] = reinterpret_cast<const uint4*>(block + kVCodes)[tid];
        s_vp[tid] = reinterpret_cast<const uint32_t*>(block + kVScale)[tid];
    }
    uint32_t out[8];
    if (mine) {
        const uint32_t sl = reinterpret_cast<const uint32_t*>(block + kKScale)[((token >> 4) * 4 + group) * 16 + (token & 15)];
        const float scale = h2f((uint16_t)sl), low = h2f((uint16_t)(sl >> 16));
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const uint32_t d = reinterpret_cast<const uint32_t*>(block)[(((token >> 4) * 4 + 2 * (part & 1) + q) * 16 + (token & 15)) * 4 + group];
#pragma unroll
            for (int e = 0; e < 8; e += 2)
                out[4 * q + e / 2] = pack_halves(__builtin_fmaf((float)((d >> nibble(e)) & 15u), scale, low),
                                                 __builtin_fmaf((float)((d >> nibble(e + 1)) & 15u), scale, low));
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
            reinterpret_cast<uint4*>(A.k_out + row)[i] = make_uint4(out[4 * i], out[4 * i + 1], out[4 * i + 2], out[4 * i + 3]);
    }
    __syncthreads();
    if (!mine) return;
    const uint16_t* vp = reinterpret_cast<const uint16_t*>(s_vp);
    const float scale = h2f(vp[group * kBlock + token]), low = h2f(vp[128 + group * kBlock + token]);
    const int e = token & 7, shift = 4 * (e / 2 + 4 * (e % 2));
    const int base = (part >> 2) * 256 + (token >> 3) * 64 + (part & 3);
#pragma unroll
    for (int n = 0; n < 16; n += 2)
        out[n / 2] = pack_halves(__builtin_fmaf((float)((s_v[base + 4 * n] >> shift) & 15u), scale, low),
                                 __builtin_fmaf((float)((s_v[base + 4 * n + 4] >> shift) & 15u), scale, low));
#pragma unroll
    for (int i = 0; i < 2; ++i)
        reinterpret_cast<uint4*>(A.v_out + row)[i] = make_uint4(out[4 * i], out[4 * i + 1], out[4 * i + 2], out[4 * i + 3]);
}

// ---------------------------------------------------------------------------
// attention of single tokens
// ---------------------------------------------------------------------------

constexpr int kWaves = 4;
// Waves at work on each SIMD.  Three of them fit with 4 query heads, and are no faster: 32 sequences of
// 16384 tokens 130 us against 124, of 2000 to 8192 tokens 38 against 37.5.
constexpr int kWavesPerSimd = 2;
constexpr int kMostWaves = 1024 * kWavesPerSimd;  // 256 CUs of 4 SIMDs
constexpr float kLog2e = 1.4426950408889634f;
// What is rounded to fp16 is a weight times a V scale, once, as an operand of the matrix cores, times the power of two
// that brings the reference of its query head and channel group to [kTop, 2 kTop).  The reference is a product so far,
// relative to the largest weight, and follows when one is more than kMost.  It follows the products, not the scales, so
// that a token of large values and no weight takes no bits from the others, and each head and group has its own: a
// product keeps fp16's eleven bits down to 2^-20 of the reference, and is lost at 2^-31.  (Scales relative to one power
// of two above all of a run's scales took 28.8 us instead of 30.7 for 8 query heads, and lost what was 2^-14 below it.)
// A power of two, as the largest weight is 1 and its products then exact, which matters where one token outweighs the
// others: with kTop / reference itself such outputs were off by 3.3e-4 instead of 2.25e-4 (2.1e-4 is their own rounding's).
// Rounding the products in two parts (22 bits) gave 2.12e-4, for 2% more time with 4 query heads and 11% with 8.
constexpr float kTop = 0x1p10f, kMost = 0x1p15f;
constexpr float kLeastReference = 0x1p-24f;  // the smallest scale: a largest weight (1) without any product needs no more
__device__ __forceinline__ float up_of(float reference) {  // kTop over the power of two not above a reference of kLeastReference or more
    return i2f((127 + 10 + 127 - (f2i(reference) >> 23)) << 23);
}
__device__ __forceinline__ float quotient(float a, float b) { return i2f(f2i(a) - f2i(b) + (127 << 23)); }  // of powers of two

// Work: a column is (sequence, KV head, set of query heads), `blocks` long; the columns lie one behind the
// other and every wave takes an equal run of blocks, across columns where it has to, so that lengths may
// differ as they like.  A wave leaves one record (maxima, sums, weighted values of its set's query heads) per
// column that it works on, at wave + column: both grow along the run, so no two share a place.
struct AttnArgs {
    Pool pool;
    const uint16_t* q;  // [B, Hq, 128]
    const int32_t* lengths;
    uint16_t* out;      // [B, Hq, 128]
    float* part;        // [records, heads of a set, 128]: weighted values
    float2* stat;       // [records, heads of a set]: maximum, sum of the weights
    int B, Hq, G, sets, columns;  // columns: of a sequence
    int waves;
    int max_length;
    float c;            // scaling * log2(e)

    __device__ __forceinline__ int blocks(int b) const { return (tokens(b) + kBlock - 1) / kBlock; }
    __device__ __forceinline__ int tokens(int b) const { return min(max(lengths[b], 0), max_length); }
};

// Blocks of a column of each sequence, summed over the sequences before b and over all.
struct Sums {
    int before, all;
};
__device__ __forceinline__ Sums sum_blocks(const AttnArgs& A, int b) {
    const int lane = lane_id();
    int before = 0, all = 0;
    for (int s = lane; s < A.B; s += kWave) {
        const int n = A.blocks(s);
        all += n;
        before += s < b ? n : 0;
    }
    return {wave_sum_int(before), wave_sum_int(all)};
}
// Blocks of a wave's run.
__device__ __forceinline__ int run_length(const AttnArgs& A, int all) { return max((all * A.columns + A.waves - 1) / A.waves, 1); }

constexpr int kPitch = kBlock + 16;  // fp32 weights of a head in the LDS: the four quarters' writes fall on different banks

// One block's codes and scalings as a lane takes them.
struct Block {
    uint4 k[2];       // tiles of 16 tokens: token lane % 16, channels 8 (lane / 16) + [0, 8) of the four groups
    uint32_t ks[2];   // scale and low of token lane % 16, group lane / 16
    uint4 v[2];       // channels 16 (4 i + j) + lane % 16 (dword j), tokens 8 (lane / 16) + [0, 8)
    uint32_t vs[4], vl[4];  // scales and lowest values of group lane % 16 / 4, tokens 8 (lane / 16) + [0, 8)
};

__device__ __forceinline__ void load_block(Block& b, const char* p, int lane) {
    const uint4* codes = reinterpret_cast<const uint4*>(p);
    b.k[0] = codes[lane];
    b.k[1] = codes[64 + lane];
    b.ks[0] = reinterpret_cast<const uint32_t*>(p + kKScale)[lane];
    b.ks[1] = reinterpret_cast<const uint32_t*>(p + kKScale)[64 + lane];
    const uint4* vc = reinterpret_cast<const uint4*>(p + kVCodes);
    b.v[0] = vc[lane];
    b.v[1] = vc[64 + lane];
    const int at = (lane & 15) / 4 * 4 + (lane >> 4);
    const uint4 s = reinterpret_cast<const uint4*>(p + kVScale)[at], l = reinterpret_cast<const uint4*>(p + kVLow)[at];
    b.vs[0] = s.x, b.vs[1] = s.y, b.vs[2] = s.z, b.vs[3] = s.w;
    b.vl[0] = l.x, b.vl[1] = l.y, b.vl[2] = l.z, b.vl[3] = l.w;
}

// One wave per workgroup; 4 HB query heads.
//
// Scores: D[row 4 g + h][token] += Q_g K^T over the four groups, where Q_g has group g's channels of
// head h in row 4 g + h and zeros elsewhere, so that lane (quarter g, token n) gets the four heads' sums over
// group g alone and applies that group's scale and lowest value (times the sum of q over the group) in fp32;
// three lane swaps add the groups and leave head h's score of token n in lane (h, n).
// Values: D[row 4 g + h][16 channels] += (P s_g) V over 32 tokens for each group's two sets of channels, the
// weights times the scale of group g in rows 4 g + h and zeros elsewhere, so that the four groups
// share one set of accumulators (32 registers otherwise, a quarter of them used).  A lane has the weights of head h in
// fp32 from the LDS, multiplies them with group g's scales, and adds up the lowest values' share in fp32 itself.
//
// The matrix cores have rows to spare (16 for 4 heads), which is why a group's place among the rows costs nothing:
// a block of 32 tokens takes 16 products, about 180 vector instructions and 5 KB.  Bound: memory for large
// batches (32 sequences of 16384 tokens, 32 / 8 heads: 119 us, 5.6 TB/s, where a kernel that only reads such pieces
// reaches 6.0), the start of a wave and the merge for small ones (1000 tokens: 4.6 + 4 us), and the chain of a block's steps
// for 8 query heads (5 sequences of 17 to 65001: 27 us, of which 17 would be memory's).
template <int HB>
__device__ __forceinline__ void work_on_column(const AttnArgs& A, float* s_p, int b, int column, int begin, int end) {
    constexpr int kHeads = 4 * HB;
    const int lane = threadIdx.x, n = lane & 15, quarter = lane >> 4;
    const int hk = column / A.sets, h0 = (column - hk * A.sets) * kHeads;  // KV head, first query head of the set within it
    const int heads = min(kHeads, A.G - h0), length = A.tokens(b);
    const long row0 = (long)b * A.Hq + hk * A.G + h0;

    // The wave's blocks, one after the other, each fetched while the one before is worked on.  Page
    // numbers come 64 at a time, one per lane.
    int entry0 = begin / A.pool.blocks, entry = 0, inside = begin - entry0 * A.pool.blocks, numbers = 0;
    auto fetch_numbers = [&]() { numbers = A.pool.table[(long)b * A.pool.width + min(entry0 + lane, A.pool.width - 1)]; };
    // next block's data, and whether its page is there
    auto fetch = [&](Block& x) {
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
    Block x0, x1;
    fetch_numbers();
    bool there0 = fetch(x0);  // before Q, so that the first block does not wait for it

    // Q: lane (n = 4 g + h, quarter): channels 32 g + 8 quarter + [0, 8) of head h, each head brought to its own
    // power of two so that the sixteenth of an element keeps its bits.  One power for all heads of the set
    // took the bits of a head whose channels are 2^-25 of another's.
    half8_t qa[HB][4];
    float qs[HB][4], back_q[HB];  // sums of a group's channels; what brings head 4 hb + quarter's scores back
    {
        const int g = n >> 2;
#pragma unroll
        for (int hb = 0; hb < HB; ++hb) {
            float x[8], top = 0.0f, sum = 0.0f;
            const int h = 4 * hb + (n & 3);
            uint4 r = {};
            if (h < heads) r = reinterpret_cast<const uint4*>(A.q + (row0 + h) * kDim)[4 * g + quarter];
            const uint32_t words[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = h2f((uint16_t)(words[e >> 1] >> (16 * (e & 1))));
                top = fmaxf(top, fabsf(x[e]));
                sum += x[e];
            }
            top = fmaxf(top, dpp<0x124>(top));  // over the groups (row_ror 4, 8) and quarters
            top = fmaxf(top, dpp<0x128>(top));
            top = swap_max(top);
            // 2^e with top * 2^e in [2^14, 2^15); 1 where there is nothing to scale, or no number
            const float up = top > 0.0f && top < INFINITY ? ldexpf(1.0f, 14 - ilogbf(top)) : 1.0f;
            sum = swap_sum16(sum, sum);
            sum = swap_sum32(sum, sum) * up * 0x1p-24f;
#pragma unroll
            for (int i = 0; i < 4; ++i) qs[hb][i] = __shfl(sum, 4 * quarter + i);
            back_q[hb] = A.c * (0x1p24f / __shfl(up, quarter));
            half8_t mine;
#pragma unroll
            for (int e = 0; e < 8; ++e) mine[e] = (_Float16)(x[e] * (e & 2 ? up * 0.0625f : up));
#pragma unroll
            for (int gg = 0; gg < 4; ++gg)
#pragma unroll
                for (int e = 0; e < 8; ++e) qa[hb][gg][e] = gg == g ? mine[e] : (_Float16)0.0f;
        }
    }

    float4_t acc[HB][2];  // channels 32 quarter + 16 i + n of the four heads, times their rows' `up`
    float m[HB], l[HB];   // head 4 hb + quarter; l: this lane's tokens
    // of row n = 4 g + h: the reference of the products; its power of two; the lowest values' share of this lane's tokens
    float reference[HB], up[HB], lows[HB];
#pragma unroll
    for (int hb = 0; hb < HB; ++hb) {
        m[hb] = -__FLT_MAX__;
        l[hb] = lows[hb] = 0.0f;
        reference[hb] = kLeastReference;
        up[hb] = up_of(kLeastReference);
#pragma unroll
        for (int i = 0; i < 2; ++i) acc[hb][i] = {0.0f, 0.0f, 0.0f, 0.0f};
    }

    auto work = [&](Block& x, int blk, bool there) {
        const int valid = there ? min(kBlock, length - blk * kBlock) : 0;
        if (valid < kBlock) {  // what lies behind the last token may be anything
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = 8 * quarter + 2 * i;
                const uint32_t keep = (t < valid ? 0xFFFFu : 0u) | (t + 1 < valid ? 0xFFFF0000u : 0u);
                x.vs[i] &= keep;
                x.vl[i] &= keep;
            }
        }
        float score[HB][2];
#pragma unroll
        for (int tile = 0; tile < 2; ++tile) {
            const uint32_t kd[4] = {x.k[tile].x, x.k[tile].y, x.k[tile].z, x.k[tile].w};
            float4_t d[HB];
#pragma unroll
            for (int hb = 0; hb < HB; ++hb) d[hb] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const half8_t kf = operand(kd[g]);
#pragma unroll
                for (int hb = 0; hb < HB; ++hb) d[hb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(qa[hb][g], kf, d[hb], 0, 0, 0);
            }
            const float scale = h2f((uint16_t)x.ks[tile]), low = h2f((uint16_t)(x.ks[tile] >> 16));
#pragma unroll
            for (int hb = 0; hb < HB; ++hb) {
                float t[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) t[i] = __builtin_fmaf(d[hb][i], scale, low * qs[hb][i]);
                const float s = swap_sum16(swap_sum32(t[0], t[2]), swap_sum32(t[1], t[3])) * back_q[hb];
                score[hb][tile] = 16 * tile + n < valid ? s : -INFINITY;
            }
        }
        bool grow = false;
#pragma unroll
        for (int hb = 0; hb < HB; ++hb) grow |= fmaxf(score[hb][0], score[hb][1]) > m[hb];
        float kept[HB];  // of row n's sums, where m moves
#pragma unroll
        for (int hb = 0; hb < HB; ++hb) kept[hb] = 1.0f;
        const bool moved = ballot(grow) != 0;
        if (moved) {
#pragma unroll
            for (int hb = 0; hb < HB; ++hb) {
                const float mn = fmaxf(m[hb], row_max16(fmaxf(score[hb][0], score[hb][1])));
                const float alpha = __builtin_amdgcn_exp2f(m[hb] - mn);
                m[hb] = mn;
                l[hb] *= alpha;
                kept[hb] = __shfl(alpha, 16 * (n & 3));
                lows[hb] *= kept[hb];
            }
        }
        // weights to LDS as [head][token]
#pragma unroll
        for (int hb = 0; hb < HB; ++hb)
#pragma unroll
            for (int tile = 0; tile < 2; ++tile) {
                const float p = __builtin_amdgcn_exp2f(score[hb][tile] - m[hb]);
                l[hb] += p;
                s_p[(4 * hb + quarter) * kPitch + 16 * tile + n] = p;
            }
        wave_sync();
        half2_t vs[4], vl[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            vs[i] = __builtin_bit_cast(half2_t, x.vs[i]);
            vl[i] = __builtin_bit_cast(half2_t, x.vl[i]);
        }
        float product[HB][8], top[HB];
        bool raise = moved;
#pragma unroll
        for (int hb = 0; hb < HB; ++hb) {
            const float4_t* const row = reinterpret_cast<const float4_t*>(&s_p[(4 * hb + (n & 3)) * kPitch + 8 * quarter]);
            const float4_t w[2] = {row[0], row[1]};
            float low[2] = {0.0f, 0.0f};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                product[hb][e] = __builtin_fmaf(w[e >> 2][e & 3], (float)vs[e >> 1][e & 1], 0.0f);
                low[e >> 2] = __builtin_fmaf(w[e >> 2][e & 3], (float)vl[e >> 1][e & 1], low[e >> 2]);
            }
            lows[hb] += low[0] + low[1];
            top[hb] = product[hb][0];
#pragma unroll
            for (int e = 1; e < 8; ++e) top[hb] = fmaxf(top[hb], product[hb][e]);
            raise |= top[hb] * up[hb] > kMost;
        }
        if (ballot(raise) != 0) {
#pragma unroll
            for (int hb = 0; hb < HB; ++hb) {
                reference[hb] = fmaxf(fmaxf(reference[hb] * kept[hb], swap_max(top[hb])), kLeastReference);
                const float next = up_of(reference[hb]), shrink = kept[hb] * quotient(next, up[hb]);
                up[hb] = next;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float a = __shfl(shrink, 4 * quarter + i);
#pragma unroll
                    for (int j = 0; j < 2; ++j) acc[hb][j][i] *= a;
                }
            }
        }
        half2_t ps[HB][4];
#pragma unroll
        for (int hb = 0; hb < HB; ++hb) {
            const float sixteenth = up[hb] * 0.0625f;  // elements 2, 3, 6, 7 meet codes times 2^-20
#pragma unroll
            for (int e = 0; e < 8; ++e)
                ps[hb][e >> 1][e & 1] = (_Float16)__builtin_fmaf(product[hb][e], e & 2 ? sixteenth : up[hb], 0.0f);  // one instruction
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const uint4& codes = x.v[g >> 1];
            const half8_t v0 = operand(g & 1 ? codes.z : codes.x), v1 = operand(g & 1 ? codes.w : codes.y);
            const uint32_t rows = (n >> 2) == g ? ~0u : 0u;
#pragma unroll
            for (int hb = 0; hb < HB; ++hb) {
                const uint4 p = __builtin_bit_cast(uint4, ps[hb]);
                const half8_t pg = __builtin_bit_cast(half8_t, make_uint4(p.x & rows, p.y & rows, p.z & rows, p.w & rows));
                acc[hb][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pg, v0, acc[hb][0], 0, 0, 0);
                acc[hb][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pg, v1, acc[hb][1], 0, 0, 0);
            }
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

    // lane (quarter g, n): channels 32 g + n and 32 g + 16 + n of the four heads
    const long record = (long)blockIdx.x + (long)b * A.columns + column;
    float* const part = A.part + record * kHeads * kDim;
#pragma unroll
    for (int hb = 0; hb < HB; ++hb) {
        const float total = row_sum16(l[hb]), sum16 = swap_sum16(lows[hb], lows[hb]), low_sum = swap_sum32(sum16, sum16);
        if (n == 0) A.stat[record * kHeads + 4 * hb + quarter] = make_float2(m[hb], total);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float low = __shfl(low_sum, 4 * quarter + i), back = __shfl(quotient(0x1p24f, up[hb]), 4 * quarter + i);
#pragma unroll
            for (int j = 0; j < 2; ++j)
                part[(4 * hb + i) * kDim + 32 * quarter + 16 * j + n] = __builtin_fmaf(acc[hb][j][i], back, low);
        }
    }
    wave_sync();
}

template <int HB>
__global__ void __launch_bounds__(kWave, kWavesPerSimd) attention_kernel(AttnArgs A) {
    constexpr int kHeads = 4 * HB;
    __shared__ __align__(16) float s_p[kHeads * kPitch];
    const int all = sum_blocks(A, 0).all, run = run_length(A, all);
    const int start = (int)blockIdx.x * run;
    int left = min(run, all * A.columns - start);
    if (left <= 0) return;
    const Item it = find_item(start / A.columns, A.B, [&](int s) { return A.blocks(s); });
    int b = it.seq;
    if (b < 0) return;
    int blocks = A.blocks(b), column = (it.index * A.columns + start % A.columns) / blocks;
    int begin = it.index * A.columns + start % A.columns - column * blocks;
    for (;;) {
        const int count = min(left, blocks - begin);
        work_on_column<HB>(A, s_p, b, column, begin, begin + count);
        left -= count;
        if (left <= 0) return;
        begin = 0;
        if (++column == A.columns) {
            column = 0;
            do {
                if (++b == A.B) return;
                blocks = A.blocks(b);
            } while (blocks == 0);
        }
    }
}

// Joins the records of a query head: PIECES workgroups per (sequence, query head), each with as many
// of its channels.  The threads take a record's maximum and sum each, and the weights from them into the LDS; the
// waves then take records' channels, two per lane, with eight loads under way, the first of them before the weights
// are known: a merge is a chain of trips to memory, of which each costs more than what it brings.  51 records
// one after the other took 28 us; 5 sequences of 17 to 65001 tokens and 32 heads, 8.4 us with one workgroup
// each and the maxima read twice, and 5.0 like this.
template <int PIECES>
__global__ void __launch_bounds__(kThreads) merge_kernel(AttnArgs A) {
    constexpr int kLanes = kWave / PIECES;     // of a record's piece: PIECES records per load
    constexpr int kStep = kWaves * PIECES;     // records that the waves take with one load
    __shared__ float2 s_record[kMostWaves];    // maximum (then weight) and sum; a wave leaves one record in a column at most
    __shared__ float2 s_o[kWaves][kLanes];
    __shared__ float s_top[kWaves], s_total[kWaves];
    const long row = blockIdx.x / PIECES;
    const int b = (int)(row / A.Hq), hq = (int)(row - (long)b * A.Hq), tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int heads = A.G <= 4 ? 4 : 8;  // of a set
    const int hk = hq / A.G, set = (hq - hk * A.G) / heads, column = hk * A.sets + set;
    const Sums sums = sum_blocks(A, b);
    const int blocks = A.blocks(b), run = run_length(A, sums.all);
    const int start = sums.before * A.columns + column * blocks, first = start / run;
    const int records = blocks == 0 ? 0 : (start + blocks - 1) / run - first + 1;
    const long at = ((long)first + (long)b * A.columns + column) * heads + (hq - hk * A.G - set * heads);
    const int of = lane / kLanes, channel = (int)blockIdx.x % PIECES * kLanes + lane % kLanes;  // record of a load, channel pair
    const float2* const stat = A.stat + at;  // a record's every `heads`
    const float2* const part = reinterpret_cast<const float2*>(A.part) + at * kWave + channel;
    uint32_t* const out = reinterpret_cast<uint32_t*>(A.out + row * kDim) + channel;
    if (records == 0) {
        if (tid < kLanes) *out = 0;
        return;
    }
    float2 r[8], o = make_float2(0.0f, 0.0f);
    auto load = [&](int i0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = part[(long)min(i0 + kStep * i + of, records - 1) * heads * kWave];
    };
    load(wave * PIECES);
    float top = -__FLT_MAX__, total = 0.0f;
    for (int s = tid; s < records; s += kThreads) {
        const float2 ml = stat[(long)s * heads];
        s_record[s] = ml;
        top = fmaxf(top, ml.x);
    }
    top = wave_max(top);
    if (lane == 0) s_top[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3]));
    for (int s = tid; s < records; s += kThreads) {
        const float2 ml = s_record[s];
        const float weight = ml.y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(ml.x - top);  // no tokens (a NaN goes on)
        s_record[s].x = weight;
        total += weight * ml.y;
    }
    total = wave_sum(total);
    if (lane == 0) s_total[wave] = total;
    __syncthreads();
    total = (s_total[0] + s_total[1]) + (s_total[2] + s_total[3]);
    for (int i0 = wave * PIECES;;) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int n = i0 + kStep * i + of;
            if (n < records) {
                const float weight = s_record[n].x;
                o.x += weight * r[i].x;
                o.y += weight * r[i].y;
            }
        }
        i0 += 8 * kStep;
        if (i0 >= records) break;
        load(i0);
    }
#pragma unroll
    for (int i = kLanes; i < kWave; i *= 2) {
        o.x += __shfl_xor(o.x, i);
        o.y += __shfl_xor(o.y, i);
    }
    if (lane < kLanes) s_o[wave][lane] = o;
    __syncthreads();
    if (tid >= kLanes) return;
#pragma unroll
    for (int i = 1; i < kWaves; ++i) {
        o.x += s_o[i][lane].x;
        o.y += s_o[i][lane].y;
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    *out = pack_halves(o.x * inv, o.y * inv);
}

// ---------------------------------------------------------------------------
// page copies
// ---------------------------------------------------------------------------

// 16 KB per workgroup through the registers.  Bound: memory, 300 pages of 32 layers (1.57 GB read and written) in
// 304 us (5.2 TB/s), 3 pages in 4 us.
constexpr int kPairs = 384;  // per launch: the numbers travel with the kernel's arguments
struct CopyArgs {
    uint4* pages;
    long pieces;  // 16-byte pieces of a page
    long layer;   // pieces of a pool
    int32_t source[kPairs], target[kPairs];
};
constexpr int kCopyPieces = 1024;  // per workgroup

__global__ void __launch_bounds__(kThreads) copy_kernel(CopyArgs A) {
    const long at = (long)blockIdx.z * A.layer + (long)blockIdx.x * kCopyPieces + threadIdx.x;
    const uint4* src = A.pages + A.source[blockIdx.y] * A.pieces + at;
    uint4* dst = A.pages + A.target[blockIdx.y] * A.pieces + at;
    const long left = A.pieces - (long)blockIdx.x * kCopyPieces - threadIdx.x;
    if (left <= 0) return;
    // (an array of uint4 would be put into the LDS here)
    const uint4 a = src[0], b = src[kThreads < left ? kThreads : 0];
    const uint4 c = src[2 * kThreads < left ? 2 * kThreads : 0], d = src[3 * kThreads < left ? 3 * kThreads : 0];
    dst[0] = a;
    if (kThreads < left) dst[kThreads] = b;
    if (2 * kThreads < left) dst[2 * kThreads] = c;
    if (3 * kThreads < left) dst[3 * kThreads] = d;
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

// Sets of query heads of a KV head: of 4, or of 8 when there are more.
int head_sets(int G) { return G <= 4 ? 1 : (G + 7) / 8; }
int set_heads(int G) { return G <= 4 ? 4 : 8; }

// Waves: as many as the chip holds at once, or one per block when there are fewer.
long attention_waves(int B, int Hk, int G, long max_length) {
    const long blocks = (max_length + kBlock - 1) / kBlock * B * Hk * head_sets(G);
    return blocks < 1 ? 1 : blocks < kMostWaves ? blocks : kMostWaves;
}
long attention_records(int B, int Hk, int G, long max_length) {
    return attention_waves(B, Hk, G, max_length) + (long)B * Hk * head_sets(G);
}

}  // namespace

extern "C" int reskv_int4_append(void* pages, int64_t num_pages, int page_tokens, int Hk, const int32_t* table,
                                 int table_width, int S, const int32_t* starts, const int32_t* offsets, const void* k,
                                 const void* v, int64_t N, const int64_t* strides, void* stream) {
    RESKV_REQUIRE(starts && k && v && strides, "null pointer");
    if (!pool_ok(pages, num_pages, page_tokens, Hk, table, table_width)) return 1;
    RESKV_REQUIRE(S > 0 && N > 0 && N < (1LL << 30) && (offsets || N == S), "bad sizes (sequences %d, rows %ld)", S, (long)N);
    RESKV_REQUIRE(aligned16(k) && aligned16(v), "rows must be 16-byte aligned");
    for (int i = 0; i < 4; ++i) RESKV_REQUIRE(strides[i] >= 0 && strides[i] % 8 == 0, "rows must be 16-byte aligned");
    const long items = row_items(offsets, S, N) * Hk;
    RESKV_REQUIRE(items < kLaunchThreads / kThreads, "too many rows or sequences");
    RowArgs A{};
    A.pool = make_pool(pages, num_pages, page_tokens, Hk, table, table_width);
    A.starts = starts;
    A.offsets = offsets;
    A.k = (const uint16_t*)k;
    A.v = (const uint16_t*)v;
    A.k_token = strides[0];
    A.k_head = strides[1];
    A.v_token = strides[2];
    A.v_head = strides[3];
    A.sequences = S;
    A.N = (int)N;
    hipLaunchKernelGGL(append_kernel<false>, dim3((unsigned)items), dim3(kThreads), 0, (hipStream_t)stream, A, Turn{});
    return reskv_host::check_launch("append_kernel");
}

extern "C" int reskv_int4_append_rope(void* pages, int64_t num_pages, int page_tokens, int Hk, const int32_t* table,
                                      int table_width, int S, const int32_t* starts, const int32_t* offsets,
                                      const int32_t* positions, const void* q, int Hq, const void* k, const void* v,
                                      int64_t N, const int64_t* strides, const float* cos, const float* sin, int rows,
                                      int rotary, int interleaved, void* q_out, int clear_rest, void* stream) {
    RESKV_REQUIRE(starts && k && v && strides && cos && sin && (!q || q_out), "null pointer");
    if (!pool_ok(pages, num_pages, page_tokens, Hk, table, table_width)) return 1;
    RESKV_REQUIRE(S > 0 && N > 0 && N < (1LL << 30) && (offsets || N == S), "bad sizes (sequences %d, rows %ld)", S, (long)N);
    RESKV_REQUIRE(!q || (Hq > 0 && Hq % Hk == 0 && Hq < (1 << 20)), "the query heads (%d) must be a multiple of the KV heads (%d)", Hq, Hk);
    RESKV_REQUIRE(rows > 0 && rotary >= 16 && rotary <= kDim && rotary % 16 == 0,
                  "the rotated channels (%d) must be a multiple of 16 up to 128, and the tables have rows", rotary);
    RESKV_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(q_out) && aligned16(cos) && aligned16(sin),
                  "tensors must be 16-byte aligned");
    for (int i = q ? 0 : 2; i < 6; ++i) RESKV_REQUIRE(strides[i] >= 0 && strides[i] % 8 == 0, "rows must be 16-byte aligned");
    const long items = row_items(offsets, S, N) * Hk;
    RESKV_REQUIRE(items < kLaunchThreads / kThreads, "too many rows or sequences");
    RowArgs A{};
    A.pool = make_pool(pages, num_pages, page_tokens, Hk, table, table_width);
    A.starts = starts;
    A.offsets = offsets;
    A.k = (const uint16_t*)k;
    A.v = (const uint16_t*)v;
    A.k_token = strides[2];
    A.k_head = strides[3];
    A.v_token = strides[4];
    A.v_head = strides[5];
    A.sequences = S;
    A.N = (int)N;
    A.clear_rest = clear_rest;
    Turn R{};
    R.q = (const uint16_t*)q;
    R.q_out = (uint16_t*)q_out;
    R.positions = positions;
    R.cos = cos;
    R.sin = sin;
    R.q_token = strides[0];
    R.q_head = strides[1];
    R.G = q ? Hq / Hk : 0;
    R.rows = rows;
    R.half = rotary / 2;
    R.interleaved = interleaved;
    const int sets = (kBlock * R.G + kQueries - 1) / kQueries;  // of a block's queries
    RESKV_REQUIRE(items * (1 + sets) < kLaunchThreads / kThreads && sets < (1 << 15), "too many rows or sequences");
    hipLaunchKernelGGL(append_kernel<true>, dim3((unsigned)items, (unsigned)(offsets || !q ? 1 + sets : 1 + (R.G + kQueries - 1) / kQueries)), dim3(kThreads), 0, (hipStream_t)stream, A, R);
    return reskv_host::check_launch("append_rope_kernel");
}

extern "C" int reskv_int4_gather(const void* pages, int64_t num_pages, int page_tokens, int Hk, const int32_t* table,
                                 int table_width, int S, const int32_t* starts, const int32_t* offsets, void* k_out,
                                 void* v_out, int64_t N, int clear_rest, void* stream) {
    RESKV_REQUIRE(starts && k_out && v_out, "null pointer");
    if (!pool_ok(pages, num_pages, page_tokens, Hk, table, table_width)) return 1;
    RESKV_REQUIRE(S > 0 && N > 0 && N < (1LL << 30) && (offsets || N == S), "bad sizes (sequences %d, rows %ld)", S, (long)N);
    RESKV_REQUIRE(aligned16(k_out) && aligned16(v_out), "rows must be 16-byte aligned");
    const long items = row_items(offsets, S, N) * Hk;
    RESKV_REQUIRE(items < kLaunchThreads / kThreads, "too many rows or sequences");
    RowArgs A{};
    A.pool = make_pool(pages, num_pages, page_tokens, Hk, table, table_width);
    A.starts = starts;
    A.offsets = offsets;
    A.k_out = (uint16_t*)k_out;
    A.v_out = (uint16_t*)v_out;
    A.sequences = S;
    A.N = (int)N;
    A.clear_rest = clear_rest;
    hipLaunchKernelGGL(gather_kernel, dim3((unsigned)items), dim3(kThreads), 0, (hipStream_t)stream, A);
    return reskv_host::check_launch("gather_kernel");
}

extern "C" int64_t reskv_int4_workspace_bytes(int B, int Hq, int Hk, int64_t max_length) {
    if (B < 1 || Hk < 1 || Hq < 1 || Hq % Hk != 0 || max_length < 0 || max_length >= (1LL << 31)) return 0;
    const int G = Hq / Hk;
    return (int64_t)attention_records(B, Hk, G, max_length) * set_heads(G) * (kDim + 2) * 4;
}

extern "C" int reskv_int4_attention(const void* q, const void* pages, int64_t num_pages, int page_tokens,
                                    const int32_t* table, int table_width, const int32_t* lengths, int B, int Hq, int Hk,
                                    float scaling, int64_t max_length, void* out, void* workspace, int64_t workspace_bytes,
                                    void* stream) {
    RESKV_REQUIRE(q && lengths && out, "null pointer");
    if (!pool_ok(pages, num_pages, page_tokens, Hk, table, table_width)) return 1;
    RESKV_REQUIRE(B > 0 && Hq > 0 && Hq % Hk == 0, "bad sizes (sequences %d, query heads %d, KV heads %d)", B, Hq, Hk);
    RESKV_REQUIRE(max_length >= 0, "max_length must not be negative");
    RESKV_REQUIRE(scaling > -1e30f && scaling < 1e30f, "scaling must lie between -1e30 and 1e30");
    RESKV_REQUIRE(aligned16(q) && aligned16(out) && aligned16(workspace), "tensors must be 16-byte aligned");
    const long most = (long)table_width * page_tokens;
    if (max_length > most) max_length = most;
    const int G = Hq / Hk;
    RESKV_REQUIRE(workspace && workspace_bytes >= reskv_int4_workspace_bytes(B, Hq, Hk, max_length), "the workspace is too small");
    const long columns = (long)Hk * head_sets(G), blocks = (max_length + kBlock - 1) / kBlock;
    // blocks, records and rows are counted in 32 bits; the last wave's run may end behind the last block
    RESKV_REQUIRE((long)B * columns * (blocks + 1) < (1L << 30) && (long)B * Hq < kLaunchThreads / kThreads,
                  "too many tokens: sequences x KV heads x blocks of %d must stay below 2^30", kBlock);
    const long records = attention_records(B, Hk, G, max_length);
    AttnArgs A{};
    A.pool = make_pool(pages, num_pages, page_tokens, Hk, table, table_width);
    A.q = (const uint16_t*)q;
    A.lengths = lengths;
    A.out = (uint16_t*)out;
    A.part = (float*)workspace;
    A.stat = (float2*)(A.part + records * set_heads(G) * kDim);
    A.B = B;
    A.Hq = Hq;
    A.G = G;
    A.sets = head_sets(G);
    A.columns = (int)columns;
    A.waves = (int)attention_waves(B, Hk, G, max_length);
    A.max_length = (int)max_length;
    A.c = scaling * kLog2e;
    hipLaunchKernelGGL(G <= 4 ? attention_kernel<1> : attention_kernel<2>, dim3((unsigned)A.waves), dim3(kWave), 0,
                       (hipStream_t)stream, A);
    if (reskv_host::check_launch("int4 attention_kernel")) return 1;
    // Query heads in pieces while there are fewer than CUs: their records come from the whole chip.  One sequence of 30000
    // tokens and 32 heads 16 us with four pieces and 20 with one, 4 of 1000 to 9000 13.6 and 14.3, 8 of them (256 heads) 18.0
    // and 17.8, 24 of 4000 35 and 28.
    const int pieces = (long)B * Hq < 256 ? 4 : 1;
    hipLaunchKernelGGL(pieces == 4 ? merge_kernel<4> : merge_kernel<1>, dim3((unsigned)(B * Hq * pieces)), dim3(kThreads), 0,
                       (hipStream_t)stream, A);
    return reskv_host::check_launch("int4 merge_kernel");
}

extern "C" int reskv_copy_pages(void* pages, int layers, int64_t num_pages, int64_t page_bytes, const int32_t* source,
                                const int32_t* target, int n, void* stream) {
    RESKV_REQUIRE(pages && source && target, "null pointer");
    RESKV_REQUIRE(layers > 0 && layers < (1 << 16) && num_pages > 0 && n >= 0 && page_bytes > 0 && page_bytes % 16 == 0,
                  "bad pool sizes (layers %d, pages %ld of %ld bytes)", layers, (long)num_pages, (long)page_bytes);
    RESKV_REQUIRE(aligned16(pages), "pages must be 16-byte aligned");
    for (int i = 0; i < n; ++i)
        RESKV_REQUIRE(source[i] >= 0 && source[i] < num_pages && target[i] >= 0 && target[i] < num_pages,
                      "page pair %d (%d to %d) is outside the pool of %ld", i, source[i], target[i], (long)num_pages);
    CopyArgs A;
    A.pages = (uint4*)pages;
    A.pieces = page_bytes / 16;
    A.layer = A.pieces * num_pages;
    const long groups = (A.pieces + kCopyPieces - 1) / kCopyPieces;
    RESKV_REQUIRE(groups < kLaunchThreads / kThreads, "pages are too large");
    for (int first = 0; first < n; first += kPairs) {
        const int count = n - first < kPairs ? n - first : kPairs;
        for (int i = 0; i < count; ++i) {
            A.source[i] = source[first + i];
            A.target[i] = target[first + i];
        }
        hipLaunchKernelGGL(copy_kernel, dim3((unsigned)groups, (unsigned)count, (unsigned)layers), dim3(kThreads), 0,
                           (hipStream_t)stream, A);
        if (reskv_host::check_launch("copy_kernel")) return 1;
    }
    return 0;
}
