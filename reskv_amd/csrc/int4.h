// Shared by the kernels of the paged 4-bit cache: where a token lies in the pool, which rows a workgroup
// has, and the operands that the matrix cores take from a block.  include/reskv_serving.h has the layout.
#pragma once

#include "serving.h"
#include "reskv_serving.h"

namespace reskv {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));

constexpr int kBlock = 32;  // tokens (>> 5 below)
constexpr int kBlockBytes = RESKV_INT4_BLOCK_BYTES;
constexpr int kKScale = 2048, kVCodes = 2560, kVScale = 4608, kVLow = 4864;  // byte offsets in a block
constexpr int kThreads = 256;

struct Pool {
    char* pages;
    const int32_t* table;  // [sequences, width]
    long num_pages;
    int blocks;  // per page
    int width, heads;

    // Block `block` of sequence s and head h, null where the table holds no page for it.
    __device__ __forceinline__ char* at(int s, int block, int h) const {
        const int entry = block / blocks;
        if (block < 0 || entry >= width) return nullptr;
        const int page = table[(long)s * width + entry];
        return in_page(page, block - entry * blocks, h);
    }
    __device__ __forceinline__ char* in_page(int page, int block, int h) const {
        if (page < 0 || page >= num_pages) return nullptr;
        return pages + (((long)page * heads + h) * blocks + block) * kBlockBytes;
    }
};

// Position of the nibble of element e = 0 .. 7 in its dword, in bits.  Elements 2 i and
// 2 i + 1 are 16 bits apart, so that one mask makes an operand register of both.
__host__ __device__ constexpr int nibble(int e) { return 4 * (e / 2 + 4 * (e % 2)); }

struct RowArgs {
    Pool pool;
    const int32_t* starts;
    const int32_t* offsets;  // null: row s is the one row of sequence s
    const uint16_t *k, *v;   // append: rows
    uint16_t *k_out, *v_out; // gather: rows [N, heads, 128]
    long k_token, k_head, v_token, v_head;  // strides of k, v in halves
    int sequences, N, clear_rest;
};

// The tokens [lo, hi) of block `block` of sequence seq that this workgroup handles, and the row of the first.
struct Part {
    int seq, block, lo, hi;
    long row;
};

__device__ __forceinline__ Part row_part(const RowArgs& A, int item) {
    if (!A.offsets) {
        const int start = A.starts[item], lead = start & (kBlock - 1);
        return {item, start >> 5, lead, lead + 1, item};
    }
    const Item it = find_item(item, A.sequences, [&](int s) {
        const int n = sequence_rows(A.offsets, s, A.N).count, lead = A.starts[s] & (kBlock - 1);
        return n == 0 ? 0 : (lead + n + kBlock - 1) / kBlock;
    });
    if (it.seq < 0) return {-1, it.index, 0, 0, 0};
    const Rows r = sequence_rows(A.offsets, it.seq, A.N);
    const int start = A.starts[it.seq], lead = start & (kBlock - 1);  // before token 0: a block without a page
    const int lo = it.index == 0 ? lead : 0, hi = min(kBlock, lead + r.count - it.index * kBlock);
    if (it.index < 0 || hi <= lo) return {-1, 0, 0, 0, 0};
    return {it.seq, (start >> 5) + it.index, lo, hi, (long)r.first + it.index * kBlock + lo - lead};
}

// Sums over lanes l and l ^ 32, l ^ 16, of two values at once.
__device__ __forceinline__ float swap_sum32(float a, float b) {
    const auto r = __builtin_amdgcn_permlane32_swap((uint32_t)f2i(a), (uint32_t)f2i(b), false, false);
    return i2f((int)r[0]) + i2f((int)r[1]);
}
__device__ __forceinline__ float swap_sum16(float a, float b) {
    const auto r = __builtin_amdgcn_permlane16_swap((uint32_t)f2i(a), (uint32_t)f2i(b), false, false);
    return i2f((int)r[0]) + i2f((int)r[1]);
}
// Maximum over the four quarters of the wave.
__device__ __forceinline__ float swap_max(float a) {
    const auto r = __builtin_amdgcn_permlane16_swap((uint32_t)f2i(a), (uint32_t)f2i(a), false, false);
    a = fmaxf(i2f((int)r[0]), i2f((int)r[1]));
    const auto s = __builtin_amdgcn_permlane32_swap((uint32_t)f2i(a), (uint32_t)f2i(a), false, false);
    return fmaxf(i2f((int)s[0]), i2f((int)s[1]));
}

// The operand register pair (elements 0 .. 7) of a dword of codes: elements 0, 1, 4, 5 times
// 2^-24 and 2, 3, 6, 7 times 2^-20.
__device__ __forceinline__ half8_t operand(uint32_t d) {
    const uint32_t e = d >> 8;
    const uint4 w = make_uint4(d & 0x000F000Fu, d & 0x00F000F0u, e & 0x000F000Fu, e & 0x00F000F0u);
    return __builtin_bit_cast(half8_t, w);
}

__device__ __forceinline__ uint32_t pack_halves(float a, float b) { return (uint32_t)f2h(a) | ((uint32_t)f2h(b) << 16); }

// Host side.

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

inline bool pool_ok(const void* pages, int64_t num_pages, int page_tokens, int Hk, const int32_t* table, int width) {
    if (!pages || !table) {
        reskv_host::set_error("null pointer");
        return false;
    }
    if (num_pages < 1 || num_pages >= (1LL << 31) || Hk < 1 || width < 1) {
        reskv_host::set_error("bad pool sizes (pages %ld, KV heads %d, table width %d)", (long)num_pages, Hk, width);
        return false;
    }
    if (page_tokens < kBlock || page_tokens % kBlock != 0 || (long)width * page_tokens >= (1L << 31)) {
        reskv_host::set_error("a page holds a multiple of %d tokens, a sequence fewer than 2^31", kBlock);
        return false;
    }
    if (!aligned16(pages)) {
        reskv_host::set_error("pages must be 16-byte aligned");
        return false;
    }
    return true;
}

inline Pool make_pool(const void* pages, int64_t num_pages, int page_tokens, int Hk, const int32_t* table, int width) {
    return Pool{(char*)pages, table, (long)num_pages, page_tokens / kBlock, width, Hk};
}

// Blocks that N rows of S sequences can touch: a sequence of n rows touches at most n / 32 + 2.
inline long row_items(const int32_t* offsets, int S, long N) { return offsets ? N / kBlock + 2L * S + 1 : (long)S; }

}  // namespace reskv
