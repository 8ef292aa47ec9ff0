// kv_cache_q4.hip -- quantising keys and values into the paged 4-bit cache as
// they are written, and reading tokens back.
//
// Scale of a block: the smallest 2^e, e in [-100, 126], with amax <= 7 * 2^e.
// With amax in (3.5, 7] units the largest value is at most one unit from its
// code (6 for everything above 5): no more than the widest step (4 to 6)
// rounds anyway, so nothing is lost to clipping and the grid is never a power
// of two coarser than it has to be.  x * 2^-e is exact, and a code is the
// nearest magnitude, ties to the even code.
//
// Bound: HBM.  A value costs 4 bytes of f32 and 17/32 of a byte in the cache.
// One lane takes eight values of a block, 4q .. 4q + 3 and 16 + 4q .. for its place q
// among the block's four lanes: each of its two loads or stores of f32 is part of 64
// bytes on end, and a block's largest magnitude is a maximum over four lanes (two DPP
// moves).  K's codes are contiguous over a wave; V's lie 16 bytes apart, the four
// tokens of a group side by side, so a workgroup takes neighbouring tokens and the L2
// merges their stores.
//
// 8192 tokens of 8 heads of 128, K and V, 76 MB each way, among other work: written and
// read back in 33.5 us; with a lane's eight values on end 35.0.  What is read back goes
// past the caches (else 36.6; alone in a loop 33.2, where this takes 34.3), what is
// written is not read past them (38.9).  Four tokens a lane with one 16-byte store of
// V's codes 39.7 (four times fewer waves in flight); workgroups of 512 or 1024 made no
// difference.  A copy of as many bytes that the last cache holds takes 10.5 each way.
#include <algorithm>

#include "q4.hpp"

namespace kore {

constexpr int kQ4Block = 256;

struct Q4Args {
    const float* in[2];  // k, v (write)
    float* out[2];       // k, v (read)
    const uint32_t* slots;
    uint8_t* cache;
    uint64_t stride[2];  // floats between two tokens of k, v
    uint32_t items;      // tokens * kv_heads * 4 nb
    uint32_t per_row, per_chunks;  // floor(2^32 / (kv_heads * 4 nb)), floor(2^32 / (4 nb))
    uint32_t head_dim;
    Q4Cache c;
};

// Integer maximum over the four lanes of a block (quad_perm 1,0,3,2 and 2,3,0,1).
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xb1, 0xf, 0xf, true));
    return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4e, 0xf, 0xf, true));
}

// i / d and i % d, inv = floor(2^32 / d): the estimate is one too small at most.
__device__ __forceinline__ uint32_t divide(uint32_t i, uint32_t d, uint32_t inv, uint32_t* rest) {
    const uint32_t q = __umulhi(i, inv), r = i - q * d;
    *rest = r >= d ? r - d : r;
    return q + (r >= d ? 1u : 0u);
}

// Item i -> token, key head, lane of the head (four a block).
__device__ __forceinline__ void q4_item(const Q4Args& a, uint32_t i, uint64_t* token, uint32_t* head, uint32_t* lane) {
    const uint32_t chunks = 4u * a.c.nb;
    uint32_t in_row;
    *token = divide(i, chunks * a.c.kv_heads, a.per_row, &in_row);
    *head = divide(in_row, chunks, a.per_chunks, lane);
}

__global__ __launch_bounds__(kQ4Block) void q4_write_kernel(Q4Args a) {
    const uint32_t i = blockIdx.x * kQ4Block + threadIdx.x;
    const int which = blockIdx.y;  // 0: K, 1: V
    if (i >= a.items) return;      // whole blocks of four lanes leave
    uint64_t token;
    uint32_t head, lane;
    q4_item(a, i, &token, &head, &lane);
    const uint32_t block = lane >> 2, q = lane & 3u;
    const float* row = a.in[which] + token * a.stride[which] + (uint64_t)head * a.head_dim;
    const uint32_t slot = a.slots[token];
    float x[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t d = 32 * block + 16 * h + 4 * q;
        if (d + 4u <= a.head_dim) {
            const f32x4 v = *reinterpret_cast<const f32x4_a4*>(row + d);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[4 * h + j] = v[j];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) x[4 * h + j] = d + j < a.head_dim ? row[d + j] : 0.0f;
        }
    }
    // The bits of |x| are ordered as their values, infinities and NaN last.
    uint32_t amax = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = max(amax, __float_as_uint(x[j]) & 0x7fffffffu);
    amax = quad_max(amax);
    const bool finite = amax < 0x7f800000u;
    // Adding the mantissa of 2 - 1.75 carries exactly where amax > 1.75 * 2^x.
    const int e = min(max((int)((amax + 0x1fffffu) >> 23) - 129, kQ4MinExp), kQ4MaxExp);
    const float unit = __uint_as_float((uint32_t)(127 + e) << 23);
    // 6 is the largest code; 3 * 2^126 the largest magnitude that the top scale holds
    // without overflow.
    const float most = fminf(6.0f * unit, __uint_as_float(0x7f400000u));
    const uint32_t page = slot >> a.c.shift, t = slot & (a.c.page - 1u);
    uint8_t* base = a.cache + (uint64_t)page * a.c.page_bytes + (uint64_t)head * a.c.head_bytes;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = __builtin_amdgcn_fmed3f(x[4 * h + j], -most, most);
        uint32_t code = 0;
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, y[0], y[1], unit, 0);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, y[2], y[3], unit, 1);
        if (!finite) code = 0;
        const uint32_t chunk = 4 * block + 2 * h + (q >> 1);
        if (page < a.c.num_pages)
            *reinterpret_cast<uint16_t*>(base + (which ? q4_v_code(a.c, t, chunk) : q4_k_code(a.c, t, chunk)) + 2 * (q & 1u)) =
                (uint16_t)code;
    }
    if (q == 0 && page < a.c.num_pages)
        base[which ? q4_v_scale(a.c, t, block) : q4_k_scale(a.c, t, block)] =
            (uint8_t)(finite ? (uint32_t)(e + 127) : kQ4NanScale);
}

__global__ __launch_bounds__(kQ4Block) void q4_read_kernel(Q4Args a) {
    const uint32_t i = blockIdx.x * kQ4Block + threadIdx.x;
    const int which = blockIdx.y;
    if (i >= a.items) return;
    uint64_t token;
    uint32_t head, lane;
    q4_item(a, i, &token, &head, &lane);
    const uint32_t block = lane >> 2, q = lane & 3u;
    const uint32_t slot = a.slots[token];
    const uint32_t page = slot >> a.c.shift, t = slot & (a.c.page - 1u);
    uint32_t code[2] = {0, 0}, b = 127;
    if (page < a.c.num_pages) {
        const uint8_t* base = a.cache + (uint64_t)page * a.c.page_bytes + (uint64_t)head * a.c.head_bytes;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t chunk = 4 * block + 2 * h + (q >> 1);
            code[h] = *reinterpret_cast<const uint16_t*>(
                base + (which ? q4_v_code(a.c, t, chunk) : q4_k_code(a.c, t, chunk)) + 2 * (q & 1u));
        }
        b = base[which ? q4_v_scale(a.c, t, block) : q4_k_scale(a.c, t, block)];
    }
    const float s = b == kQ4NanScale ? __uint_as_float(0x7fc00000u) : q4_scale(b);
    float* row = a.out[which] + (token * a.c.kv_heads + head) * a.head_dim;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t d = 32 * block + 16 * h + 4 * q;
        const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code[h], 1.0f, 0);
        const auto hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code[h], 1.0f, 1);
        const f32x4 v = {lo[0] * s, lo[1] * s, hi[0] * s, hi[1] * s};
        if (d + 4u <= a.head_dim) {
            __builtin_nontemporal_store((f32x4_a4)v, reinterpret_cast<f32x4_a4*>(row + d));
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (d + j < a.head_dim) row[d + j] = v[j];
        }
    }
}

static bool overlap(const void* a, uint64_t na, const void* b, uint64_t nb) {
    const char *p = (const char*)a, *q = (const char*)b;
    return p < q + nb && q < p + na;
}

// Tokens in bands: a launch holds fewer than 2^32 threads.
template <typename Kernel>
static int q4_launch(Kernel kernel, Q4Args a, uint64_t tokens, bool write, hipStream_t s) {
    const uint64_t per_token = (uint64_t)a.c.kv_heads * 4u * a.c.nb;
    a.per_row = (uint32_t)((1ull << 32) / per_token);
    a.per_chunks = (uint32_t)((1ull << 32) / (4u * a.c.nb));
    const uint64_t band = std::max<uint64_t>(1, (1ull << 30) / per_token);
    for (uint64_t t = 0; t < tokens; t += band) {
        const uint64_t n = std::min(band, tokens - t);
        a.items = (uint32_t)(n * per_token);
        hipLaunchKernelGGL(kernel, dim3((a.items + kQ4Block - 1) / kQ4Block, 2), dim3(kQ4Block), 0, s, a);
        const int st = launch_status();
        if (st != KORE_HIP_OK) return st;
        a.slots += n;
        for (int w = 0; w < 2; ++w) {
            if (write) a.in[w] += n * a.stride[w];
            else a.out[w] += n * (uint64_t)a.c.kv_heads * a.head_dim;
        }
    }
    return KORE_HIP_OK;
}

}  // namespace kore

using namespace kore;

extern "C" uint64_t kore_hip_kv_cache_q4_bytes(uint64_t num_pages, uint64_t page_size, uint64_t kv_heads,
                                               uint64_t head_dim) {
    Q4Cache c;
    uint64_t bytes;
    return q4_layout(num_pages, page_size, kv_heads, head_dim, &c, &bytes) == KORE_HIP_OK ? bytes : 0;
}

extern "C" int kore_hip_kv_cache_write_q4_f32(const float* k, const float* v, const uint32_t* slots, uint8_t* cache,
                                              uint64_t tokens, uint64_t kv_heads, uint64_t head_dim,
                                              uint64_t num_pages, uint64_t page_size, uint64_t k_stride,
                                              uint64_t v_stride, kore_stream_t stream) {
    if (tokens == 0 || kv_heads == 0 || head_dim == 0 || num_pages == 0) return KORE_HIP_OK;
    Q4Args a = {};
    uint64_t bytes, span[2];
    const int st = q4_layout(num_pages, page_size, kv_heads, head_dim, &a.c, &bytes);
    if (st != KORE_HIP_OK) return st;
    if (!k || !v || !slots || !cache) return KORE_HIP_ERR_NULL_PTR;
    if (!aligned16(cache)) return KORE_HIP_ERR_BAD_DIM;
    const uint64_t row = kv_heads * head_dim;
    a.stride[0] = k_stride ? k_stride : row;
    a.stride[1] = v_stride ? v_stride : row;
    for (int w = 0; w < 2; ++w) {
        if (a.stride[w] < row) return KORE_HIP_ERR_BAD_DIM;
        if (!mul_ok(tokens, a.stride[w], &span[w]) || span[w] > kMaxElements) return KORE_HIP_ERR_OVERFLOW;
        span[w] = ((tokens - 1) * a.stride[w] + row) * 4;
    }
    if (overlap(cache, bytes, k, span[0]) || overlap(cache, bytes, v, span[1]) ||
        overlap(cache, bytes, slots, tokens * 4))
        return KORE_HIP_ERR_ALIAS;
    a.in[0] = k;
    a.in[1] = v;
    a.slots = slots;
    a.cache = cache;
    a.head_dim = (uint32_t)head_dim;
    return q4_launch(q4_write_kernel, a, tokens, true, (hipStream_t)stream);
}

extern "C" int kore_hip_kv_cache_read_q4_f32(const uint8_t* cache, const uint32_t* slots, float* k_out, float* v_out,
                                             uint64_t tokens, uint64_t kv_heads, uint64_t head_dim,
                                             uint64_t num_pages, uint64_t page_size, kore_stream_t stream) {
    if (tokens == 0 || kv_heads == 0 || head_dim == 0) return KORE_HIP_OK;
    Q4Args a = {};
    uint64_t bytes, elems;
    const int st = q4_layout(num_pages, page_size, kv_heads, head_dim, &a.c, &bytes);
    if (st != KORE_HIP_OK) return st;
    if (!slots || !k_out || !v_out || (num_pages && !cache)) return KORE_HIP_ERR_NULL_PTR;
    if (num_pages && !aligned16(cache)) return KORE_HIP_ERR_BAD_DIM;
    if (!mul_ok(tokens, kv_heads * head_dim, &elems) || elems > kMaxElements) return KORE_HIP_ERR_OVERFLOW;
    if (overlap(k_out, elems * 4, v_out, elems * 4) || overlap(cache, bytes, k_out, elems * 4) ||
        overlap(cache, bytes, v_out, elems * 4) || overlap(slots, tokens * 4, k_out, elems * 4) ||
        overlap(slots, tokens * 4, v_out, elems * 4))
        return KORE_HIP_ERR_ALIAS;
    a.out[0] = k_out;
    a.out[1] = v_out;
    a.slots = slots;
    a.cache = const_cast<uint8_t*>(cache);
    a.head_dim = (uint32_t)head_dim;
    return q4_launch(q4_read_kernel, a, tokens, false, (hipStream_t)stream);
}
