// q4.hpp -- the paged 4-bit key/value cache: layout and codes.
//
// A block is 32 consecutive values of one token's head: 32 E2M1 codes (sign, 2
// exponent bits, 1 mantissa bit; magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6) and one
// scale byte b, the power of two 2^(b - 127), or NaN for b = 255.  17 bytes for
// 32 values.  gfx950 turns two codes and their scale into two bf16 values in
// one instruction, and the product of a code and a power of two is exact in
// bf16: the cache's values are matrix operands as they are.
//
// Bytes of one page of one key head (P tokens, nb = ceil(head_dim / 32)):
//   K codes   [P][16 nb]       dimension 2j in the low half of byte j
//   V codes   [P / 16][4 g][4 nb chunks][4 i][4 bytes]
//             token 4 g + i of the 16, chunk c = dimensions 8c .. 8c + 7
//   K scales  [P][nb]
//   V scales  [P / 16][nb][16 tokens]
// K's rows are what a lane of the score product reads: 16 tokens x 4 groups of
// dimensions, 16 bytes a lane.  V is reduced over tokens, so a lane of the value
// product wants several tokens of the same dimensions: four tokens x eight
// dimensions lie in 16 consecutive bytes, and a 16-token tile of either operand
// is one contiguous kilobyte at head_dim 128.
#pragma once

#include "common.hpp"
#include "kore_hip_internal.hpp"

namespace kore {

constexpr uint32_t kQ4MaxHeadDim = 256;
constexpr uint32_t kQ4MaxPage = 65536;
constexpr int kQ4MinExp = -100;  // scales of 2^-100 and more
constexpr int kQ4MaxExp = 126;
constexpr uint32_t kQ4NanScale = 255;

struct Q4Cache {
    uint64_t page_bytes;  // all key heads of a page
    uint32_t head_bytes;  // one key head of a page
    uint32_t nb;          // blocks of 32 values in a head
    uint32_t page;        // tokens in a page
    uint32_t shift;       // log2(page)
    uint32_t kv_heads;
    uint32_t num_pages;
};

// Checks the cache's dimensions; bytes: its whole size.
inline int q4_layout(uint64_t num_pages, uint64_t page_size, uint64_t kv_heads, uint64_t head_dim, Q4Cache* c,
                     uint64_t* bytes) {
    if (head_dim == 0 || head_dim > kQ4MaxHeadDim || page_size < 16 || page_size > kQ4MaxPage ||
        (page_size & (page_size - 1)))
        return KORE_HIP_ERR_BAD_DIM;
    if (kv_heads > 65535u || num_pages > 0xffffffffull) return KORE_HIP_ERR_OVERFLOW;
    c->nb = (uint32_t)((head_dim + 31) / 32);
    c->page = (uint32_t)page_size;
    c->shift = (uint32_t)__builtin_ctzll(page_size);
    c->head_bytes = c->page * c->nb * 34u;
    c->kv_heads = (uint32_t)kv_heads;
    c->num_pages = (uint32_t)num_pages;
    c->page_bytes = (uint64_t)c->head_bytes * kv_heads;
    if (!mul_ok(c->page_bytes, num_pages, bytes) || *bytes > kMaxElements) return KORE_HIP_ERR_OVERFLOW;
    return KORE_HIP_OK;
}

// Byte offsets inside one page of one key head, for token t of the page.
__device__ __forceinline__ uint32_t q4_k_code(const Q4Cache& c, uint32_t t, uint32_t chunk) {
    return t * c.nb * 16u + chunk * 4u;
}
__device__ __forceinline__ uint32_t q4_v_code(const Q4Cache& c, uint32_t t, uint32_t chunk) {
    return c.page * c.nb * 16u + ((((t >> 4) * 4u + ((t >> 2) & 3u)) * 4u * c.nb + chunk) * 4u + (t & 3u)) * 4u;
}
__device__ __forceinline__ uint32_t q4_k_scale(const Q4Cache& c, uint32_t t, uint32_t block) {
    return c.page * c.nb * 32u + t * c.nb + block;
}
__device__ __forceinline__ uint32_t q4_v_scale(const Q4Cache& c, uint32_t t, uint32_t block) {
    return c.page * c.nb * 33u + ((t >> 4) * c.nb + block) * 16u + (t & 15u);
}

// 2^(b - 127); 2^-127 is subnormal.
__device__ __forceinline__ float q4_scale(uint32_t b) {
    return __uint_as_float(b ? b << 23 : 0x00400000u);
}

}  // namespace kore
