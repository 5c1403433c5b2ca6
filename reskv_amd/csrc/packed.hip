// Causal attention of packed sequences of different lengths (include/reskv_serving.h).
//
// One workgroup of four waves per 128 rows of one KV head and sequence, where row r is
// query r / G of query head r % G of the head's group: short sequences and single tokens then fill
// the matrix cores' columns with the heads of a group, whatever G is.  A wave owns 32
// rows; keys are taken 64 at a time from double-buffered LDS.
//   S^T = K Q^T on v_mfma_f32_32x32x16_f16: lane (col = lane % 32, half = lane / 32)
//     holds its row's scores of keys 8 (i / 4) + 4 half + i % 4, i = 0..15, of a
//     32-key block, so the softmax needs one lane swap, and the fp16 weights are the
//     B operand of
//   O^T = V^T P^T as they are: its 16-key steps take the keys in the order in which
//     a lane holds them, and V^T comes from the staged rows through LDS transpose
//     reads of the same keys.
// Scores, softmax and sums are fp32.  The weights are rounded to fp16 for the second product;
// they are 2^14 exp2(x - m), so that a weight is lost only when it is below 2^-39 of the
// largest.
#include "serving.h"
#include "reskv_serving.h"

using namespace reskv;

namespace {

typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float16_t __attribute__((ext_vector_type(16)));
typedef short short4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) short4_t lds_short4_t;

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kWaveRows = 32;
constexpr int kRows = kWaves * kWaveRows;
constexpr int kKeys = 64;         // keys per tile
constexpr int kPitch = kDim + 8;  // halves per staged row (16-byte aligned, rows start on different banks)
constexpr int kTileHalves = kKeys * kPitch;
constexpr int kPieces = kKeys * kDim / 8 / kThreads;  // 16-byte pieces of a K (or V) tile per thread
constexpr float kWeightBits = 14.0f;
constexpr int kRecord = kDim + 2;

struct PackedArgs {
    const uint16_t *q, *k, *v;
    uint16_t* out;               // [Nq, Hq, 128]
    const int32_t *q_offsets, *k_offsets;
    float* part;                 // [splits, Nq * Hq, 130]: o[128], m, l
    long q_token, q_head, k_token, k_head, v_token, v_head;  // strides in halves
    int sequences, Nq, Nk, Hq, Hk, G;
    int items, splits, clear_rest;
    float c;                     // scaling * log2(e)
};

__device__ __forceinline__ bool not_finite(uint32_t pair) {
    return ((pair & 0x7C00u) == 0x7C00u) || ((pair & 0x7C000000u) == 0x7C000000u);
}
__device__ __forceinline__ uint32_t finite_or_zero(uint32_t pair) {
    return pair & (((pair & 0x7C00u) == 0x7C00u ? 0u : 0xFFFFu) | ((pair & 0x7C000000u) == 0x7C000000u ? 0u : 0xFFFF0000u));
}

__global__ void __launch_bounds__(kThreads, 2) packed_kernel(PackedArgs A) {
    __shared__ __align__(16) uint16_t s_kv[2][2][kTileHalves];  // [buffer][K, V]
    __shared__ int s_odd[2];  // the last tile on the diagonal whose V held a value that is not finite, per buffer
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, half = lane >> 5;
    // the KV heads take turns, so that a head's workgroups share an XCD's L2 when there are
    // 8 heads; the last sequence and a sequence's last rows, which see most keys, come first
    int w = blockIdx.x;
    const int hk = w % A.Hk;
    w /= A.Hk;
    const int split = w % A.splits, item = A.items - 1 - w / A.splits;
    const Item it = find_item(item, A.sequences, [&](int s) {
        return (int)(((long)sequence_rows(A.q_offsets, s, A.Nq).count * A.G + kRows - 1) / kRows);
    });
    if (it.seq < 0) {
        // behind the last item (there is always one such): rows of no sequence
        if (A.clear_rest && split == 0) {
            const int begin = min(max(A.q_offsets[0], 0), A.Nq);
            const int end = min(max(A.q_offsets[A.sequences], begin), A.Nq);
            const int spares = A.items - (item - it.index), rest = begin + A.Nq - end;
            const int per_row = A.G * 16;  // 16-byte pieces of a query's heads in the group
            for (long i = (long)it.index * kThreads + tid; i < (long)rest * per_row; i += (long)spares * kThreads) {
                const int r = (int)(i / per_row), at = (int)(i - (long)r * per_row);
                const long row = r < begin ? r : end + r - begin;
                reinterpret_cast<uint4*>(A.out + (row * A.Hq + (long)hk * A.G) * kDim)[at] = make_uint4(0, 0, 0, 0);
            }
        }
        return;
    }
    const Rows qr = sequence_rows(A.q_offsets, it.seq, A.Nq), kr = sequence_rows(A.k_offsets, it.seq, A.Nk);
    const int nq = qr.count, nk = kr.count, ahead = nk - nq;  // query i sees keys up to i + ahead
    const long rows = (long)nq * A.G;
    const long r0 = (long)it.index * kRows + wave * kWaveRows;  // the wave's first row
    if (it.index < 0 || (long)it.index * kRows >= rows) return;
    const long r = min(r0 + col, rows - 1);
    const int query = (int)(r / A.G), head = hk * A.G + (int)(r - (long)query * A.G);
    const int sees = min(query + ahead + 1, nk);  // keys that this lane's row sees; none when not positive
    // keys that some row of the wave sees, and that all of them see
    const int wave_last = min((int)(min(r0 + kWaveRows, rows) - 1) / A.G + ahead + 1, nk);
    const int wave_all = r0 < rows ? (int)(r0 / A.G) + ahead + 1 : 0;
    const int wave_any = r0 < rows ? wave_last : 0;
    const int group_last = min((int)((min((long)(it.index + 1) * kRows, rows) - 1) / A.G) + ahead + 1, nk);
    const int group_all = (int)((long)it.index * kRows / A.G) + ahead + 1;
    const int tiles = group_last > 0 ? (group_last + kKeys - 1) / kKeys : 0;
    const int per_split = (tiles + A.splits - 1) / A.splits;
    const int tile0 = split * per_split, tile1 = min(tile0 + per_split, tiles);

    // Q operand: lane (col, half) holds its row, channels 16 kk + 8 half + [0, 8)
    half8_t qf[8];
    {
        const uint4* src = reinterpret_cast<const uint4*>(A.q + (qr.first + query) * A.q_token + head * A.q_head);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) qf[kk] = __builtin_bit_cast(half8_t, src[2 * kk + half]);
    }

    // Tiles are fetched through range-checked buffer loads without branches: a row behind the
    // sequence's last key has an offset behind the resource's end and comes as zeros.
    const uint16_t* kb = A.k + kr.first * A.k_token + hk * A.k_head;
    const uint16_t* vb = A.v + kr.first * A.v_token + hk * A.v_head;
    constexpr int kEnd = 0x40000000;
    uint4 kreg[kPieces], vreg[kPieces];
    auto fetch = [&](int tile) {
        const __amdgpu_buffer_rsrc_t kres =
            __builtin_amdgcn_make_buffer_rsrc((void*)(kb + (long)tile * kKeys * A.k_token), 0, kEnd, 0x00020000);
        const __amdgpu_buffer_rsrc_t vres =
            __builtin_amdgcn_make_buffer_rsrc((void*)(vb + (long)tile * kKeys * A.v_token), 0, kEnd, 0x00020000);
        const int left = nk - tile * kKeys;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int p = tid + kThreads * i, row = p >> 4, at = 16 * (p & 15);
            const int ko = row < left ? row * (int)A.k_token * 2 + at : kEnd;
            const int vo = row < left ? row * (int)A.v_token * 2 + at : kEnd;
            kreg[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(kres, ko, 0, 0));
            vreg[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(vres, vo, 0, 0));
        }
    };
    // A key that a row does not see has weight 0, and its value must not matter to the row, also
    // when it is infinite or NaN: in the tiles on the diagonal such values are staged as zeros
    // and added to the rows that see them apart.
    auto stage = [&](int buf, int tile) {
        if ((tile + 1) * kKeys > group_all) {
            bool odd = false;
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                odd = odd || not_finite(vreg[i].x) || not_finite(vreg[i].y) || not_finite(vreg[i].z) || not_finite(vreg[i].w);
                vreg[i] = make_uint4(finite_or_zero(vreg[i].x), finite_or_zero(vreg[i].y), finite_or_zero(vreg[i].z),
                                     finite_or_zero(vreg[i].w));
            }
            if (odd) s_odd[buf] = tile;
        }
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int p = tid + kThreads * i;
            const int at = (p >> 4) * kPitch + 8 * (p & 15);
            *reinterpret_cast<uint4*>(&s_kv[buf][0][at]) = kreg[i];
            *reinterpret_cast<uint4*>(&s_kv[buf][1][at]) = vreg[i];
        }
    };

    float16_t acc[4];  // O^T: channels 32 db + 8 (i / 4) + 4 half + i % 4 of the lane's row
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[db][i] = 0.0f;
    // log2-domain maximum, and this lane's half of the weights' sum.  The maximum starts at
    // the lowest finite value: scores of minus infinity then weigh exp2(-inf) = 0, where
    // against a maximum of minus infinity they would give NaN
    float m = -__FLT_MAX__, l = 0.0f;
    // transpose reads: lane i of a 16-lane row points at key i / 4, channel 4 (i % 4) of
    // its 4 x 16 block and receives the block's four keys of channel i
    const int i16 = lane & 15;
    const int vt = (4 * half + (i16 >> 2)) * kPitch + 16 * ((lane >> 4) & 1) + 4 * (i16 & 3);

    if (tid < 2) s_odd[tid] = -1;
    __syncthreads();
    if (tile0 < tile1) {
        fetch(tile0);
        stage(tile0 & 1, tile0);
    }
    __syncthreads();
    for (int tile = tile0; tile < tile1; ++tile) {
        const int buf = tile & 1, base = tile * kKeys;
        fetch(tile + 1);
        if (base < wave_any) {  // wave-uniform: a tile that no row of the wave sees is left out
            const uint16_t* sk = s_kv[buf][0];
            const uint16_t* sv = s_kv[buf][1];
            float16_t s[2];
#pragma unroll
            for (int kb2 = 0; kb2 < 2; ++kb2) {
#pragma unroll
                for (int i = 0; i < 16; ++i) s[kb2][i] = 0.0f;
#pragma unroll
                for (int kk = 0; kk < 8; ++kk) {
                    const half8_t kf = *reinterpret_cast<const half8_t*>(sk + (32 * kb2 + col) * kPitch + 16 * kk + 8 * half);
                    s[kb2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[kk], s[kb2], 0, 0, 0);
                }
            }
            if (base + kKeys > wave_all) {  // the diagonal
#pragma unroll
                for (int kb2 = 0; kb2 < 2; ++kb2)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (base + 32 * kb2 + 8 * (i >> 2) + 4 * half + (i & 3) >= sees) s[kb2][i] = -INFINITY;
            }
            float mx = s[0][0];
#pragma unroll
            for (int kb2 = 0; kb2 < 2; ++kb2)
#pragma unroll
                for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[kb2][i]);
            const auto sw = __builtin_amdgcn_permlane32_swap((uint32_t)f2i(mx), (uint32_t)f2i(mx), false, false);
            mx = fmaxf(i2f((int)sw[0]), i2f((int)sw[1])) * A.c;  // c > 0
            if (ballot(mx > m) != 0) {
                const float mn = fmaxf(m, mx);
                const float alpha = __builtin_amdgcn_exp2f(m - mn);
                m = mn;
                l *= alpha;
#pragma unroll
                for (int db = 0; db < 4; ++db)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[db][i] *= alpha;
            }
            half8_t pf[4];  // the weights of 16-key steps, keys in the lane's order
            float sum = 0.0f;
            const float shift = kWeightBits - m;
#pragma unroll
            for (int kb2 = 0; kb2 < 2; ++kb2)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb2][i], A.c, shift));
                    sum += p;
                    pf[2 * kb2 + (i >> 3)][i & 7] = (_Float16)p;
                }
            l += sum;
#pragma unroll
            for (int st = 0; st < 4; ++st)
#pragma unroll
                for (int db = 0; db < 4; ++db) {
                    const uint16_t* src = sv + vt + 16 * st * kPitch + 32 * db;
                    const half4_t lo = __builtin_bit_cast(half4_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t*)src));
                    const half4_t hi = __builtin_bit_cast(
                        half4_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t*)(src + 8 * kPitch)));
                    const half8_t vf = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                    acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pf[st], acc[db], 0, 0, 0);
                }
            if (s_odd[buf] == tile) {  // rare: what was staged as zero, to the rows that see it
                const int last = min(base + kKeys, nk);
                for (int j = base; j < last; ++j) {
                    const uint16_t* row = vb + (long)j * A.v_token;
#pragma unroll
                    for (int db = 0; db < 4; ++db)
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float x = h2f(row[32 * db + 8 * (i >> 2) + 4 * half + (i & 3)]);
                            if (j < sees && !(fabsf(x) < INFINITY)) acc[db][i] += x;
                        }
                }
            }
        }
        if (tile + 1 < tile1) stage(buf ^ 1, tile + 1);  // last read in the tile before, which a barrier ended
        __syncthreads();
    }

    const auto ls = __builtin_amdgcn_permlane32_swap((uint32_t)f2i(l), (uint32_t)f2i(l), false, false);
    const float total = i2f((int)ls[0]) + i2f((int)ls[1]);
    if (r0 + col >= rows) return;
    const long row = ((long)qr.first + query) * A.Hq + head;
    if (A.splits > 1) {
        float* rec = A.part + ((long)split * A.Nq * A.Hq + row) * kRecord;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int i = 0; i < 16; i += 2)
                *reinterpret_cast<float2*>(rec + 32 * db + 8 * (i >> 2) + 4 * half + (i & 3)) = make_float2(acc[db][i], acc[db][i + 1]);
        if (half == 0) *reinterpret_cast<float2*>(rec + kDim) = make_float2(m, total);
        return;
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    uint16_t* dst = A.out + row * kDim;
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t word[2];
#pragma unroll
            for (int e = 0; e < 2; ++e)
                word[e] = (uint32_t)f2h(acc[db][4 * j + 2 * e] * inv) | ((uint32_t)f2h(acc[db][4 * j + 2 * e + 1] * inv) << 16);
            *reinterpret_cast<uint2*>(dst + 32 * db + 8 * j + 4 * half) = make_uint2(word[0], word[1]);
        }
}

// Joins the splits: one wave per (query, head) row, two channels per lane.  Rows of no
// sequence have no records and are left to the attention's own workgroups.
__global__ void __launch_bounds__(kThreads) packed_merge_kernel(PackedArgs A) {
    const int lane = threadIdx.x & 63;
    const long row = (long)blockIdx.x * kWaves + (threadIdx.x >> 6), all = (long)A.Nq * A.Hq;
    if (row >= all) return;
    const int query = (int)(row / A.Hq);
    if (query < A.q_offsets[0] || query >= A.q_offsets[A.sequences]) return;
    float top = -__FLT_MAX__;
    for (int s = 0; s < A.splits; ++s) top = fmaxf(top, A.part[(s * all + row) * kRecord + kDim]);
    float o0 = 0.0f, o1 = 0.0f, total = 0.0f;
    for (int s = 0; s < A.splits; ++s) {
        const float* rec = A.part + (s * all + row) * kRecord;
        const float l = rec[kDim + 1];
        if (l == 0.0f) continue;  // no keys (a NaN goes on)
        const float a = __builtin_amdgcn_exp2f(rec[kDim] - top);
        const float2 o = reinterpret_cast<const float2*>(rec)[lane];
        o0 += a * o.x;
        o1 += a * o.y;
        total += a * l;
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    reinterpret_cast<uint32_t*>(A.out + row * kDim)[lane] = (uint32_t)f2h(o0 * inv) | ((uint32_t)f2h(o1 * inv) << 16);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

// Tiles of 128 rows that S sequences of Nq rows in all can bring, and one that is always free.
long packed_items(int S, long Nq, int G) { return Nq * G / kRows + S + 1; }

// Splits of the keys: none while the rows alone give every CU its two workgroups, else up to as
// many as do, of at least 512 keys each.
int packed_splits(int S, long Nq, int Hk, int G, long max_keys) {
    const long groups = packed_items(S, Nq, G) * Hk;
    long splits = 512 / groups;
    if (splits > max_keys / 512) splits = max_keys / 512;
    return splits < 1 ? 1 : (int)splits;
}

}  // namespace

extern "C" int64_t reskv_packed_workspace_bytes(int S, int64_t Nq, int Hq, int Hk, int64_t max_keys) {
    if (S < 1 || Nq < 1 || Hk < 1 || Hq < 1 || Hq % Hk != 0) return 0;
    const int splits = packed_splits(S, Nq, Hk, Hq / Hk, max_keys);
    return splits == 1 ? 0 : (int64_t)splits * Nq * Hq * kRecord * 4;
}

extern "C" int reskv_packed_attention(const void* q, const void* k, const void* v, void* out, const int32_t* q_offsets,
                                      const int32_t* k_offsets, int S, int64_t Nq, int64_t Nk, int Hq, int Hk,
                                      const int64_t* strides, float scaling, int64_t max_keys, int clear_rest,
                                      void* workspace, int64_t workspace_bytes, void* stream) {
    RESKV_REQUIRE(q && k && v && out && q_offsets && k_offsets && strides, "null pointer");
    RESKV_REQUIRE(S > 0 && Nq > 0 && Nk > 0 && Hk > 0 && Hq > 0 && Hq % Hk == 0,
                  "bad sizes (sequences %d, Nq %ld, Nk %ld, Hq %d, Hk %d)", S, (long)Nq, (long)Nk, Hq, Hk);
    const int G = Hq / Hk;
    RESKV_REQUIRE(Nq < (1LL << 30) && Nk < (1LL << 30), "too many rows");
    RESKV_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out), "tensors must be 16-byte aligned");
    for (int i = 0; i < 6; ++i) RESKV_REQUIRE(strides[i] >= 0 && strides[i] % 8 == 0, "rows must be 16-byte aligned");
    RESKV_REQUIRE(strides[2] < (1 << 23) && strides[4] < (1 << 23), "token strides of k and v must be below 2^23");
    RESKV_REQUIRE(scaling > 0.0f, "scaling must be positive");
    const int splits = packed_splits(S, Nq, Hk, G, max_keys);
    RESKV_REQUIRE(splits == 1 || (workspace && workspace_bytes >= reskv_packed_workspace_bytes(S, Nq, Hq, Hk, max_keys)),
                  "the workspace is too small");
    PackedArgs A{};
    A.q = (const uint16_t*)q;
    A.k = (const uint16_t*)k;
    A.v = (const uint16_t*)v;
    A.out = (uint16_t*)out;
    A.q_offsets = q_offsets;
    A.k_offsets = k_offsets;
    A.part = (float*)workspace;
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
    RESKV_REQUIRE(items * Hk * splits < (1L << 31), "too many rows");
    A.items = (int)items;
    A.splits = splits;
    A.clear_rest = clear_rest;
    A.c = scaling * 1.4426950408889634f;
    hipLaunchKernelGGL(packed_kernel, dim3((unsigned)(items * Hk * splits)), dim3(kThreads), 0, (hipStream_t)stream, A);
    if (reskv_host::check_launch("packed_kernel")) return 1;
    if (splits == 1) return 0;
    const long rows = (long)Nq * Hq;
    hipLaunchKernelGGL(packed_merge_kernel, dim3((unsigned)((rows + kWaves - 1) / kWaves)), dim3(kThreads), 0,
                       (hipStream_t)stream, A);
    return reskv_host::check_launch("packed_merge_kernel");
}
