// attention_q4.hip -- softmax(scale q k^T) v over the paged 4-bit cache, for
// ragged sequences with any number of new tokens each.
//
// One pass over the keys with the running maximum and sum of the softmax; no
// scores in memory.  The rows of one key head are its query heads times the
// sequence's new tokens: row r = token * group + head, 16 to a matrix tile.
//
// Arithmetic.  A cached value is a code times a power of two, exact in bf16, and
// gfx950 makes two of them with their scale in one instruction, so the matrix
// cores' bf16 form loses nothing on the cache's side.  A query value (times scale
// * log2 e, one f32 rounding) is cut into three bf16 terms of 8 bits each, which
// is all of its 24: every product q * k is exact and sums are f32.  A probability
// is two bf16 terms rounded to nearest: it is off by at most 2^-18 of itself, next
// to the few f32 roundings of the score that it is the exponential of; the row's
// sum takes the f32 value.
// (The block-scaled product takes K's codes and scales as they lie, and q as six
// E4M3 terms; but its sum keeps only some 2^-19 of the largest product, so blocks
// of very different scales would cost accuracy that f32 has.)
//
// Layout of a step (32 tokens; n = lane % 16, g = lane / 16):
//   S^T = K Q^T   a lane holds token n's dimensions of group g (K's codes as
//                 they lie, 16 bytes at head_dim 128) and row n's same
//                 dimensions: which eight of them meet in one product is free.
//                 It gets tokens 4g .. 4g + 3 of row n.
//   O^T = V^T P^T the operand P^T wants eight tokens of row n from lane group g:
//                 the four it has of this 16-token tile and the four of the
//                 next.  V's operand is taken in the same order of tokens, so P
//                 moves between no lanes and through no memory.
// All of a lane's values belong to row n: maximum, sum and rescaling are its
// own, but for a maximum over the four lane groups.
//
// A masked token's score is -inf whatever its codes say.  Its V is finite (the
// scale of a token past the cache's length counts as 1); where V of a token
// that only later rows see is NaN, the product uses 1 for the scale and the
// rows that see it are set to NaN one by one.
#include <algorithm>
#include <type_traits>

#include "q4.hpp"

namespace kore {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kAttBlock = 256;
constexpr int kAttWaves = kAttBlock / kWave;
constexpr uint32_t kAttStep = 32;      // tokens of a step
constexpr uint32_t kAttMinChunk = 8;   // steps of a split, at least
constexpr uint32_t kAttMaxSteps = 1u << 27;  // more than 2^31 keys have
constexpr int kAttTerms = 3;           // bf16 terms of a query value
constexpr uint32_t kAttJoin = 512;  // threads of the joining kernel
constexpr uint32_t kAttMaxSplits = 1024;

struct AttArgs {
    const float* q;
    const uint8_t* cache;
    const uint32_t* table;   // [num_seqs][max_pages]
    const uint32_t* lens;    // [num_seqs]
    const uint32_t* starts;  // [num_seqs + 1]
    float* out;
    float* part;
    uint64_t q_stride;
    uint64_t tokens;
    uint32_t num_seqs, q_heads, group, max_pages, dim;
    uint32_t items, item0;  // work items there can be (see att_item), first of this launch
    uint32_t target;        // items to cut the keys into, 0: one a tile
    float scale_log2;
    int causal;
    Q4Cache c;
};

// A work item: kRows consecutive rows of one sequence and one share of its keys.
struct AttItem {
    uint32_t seq, q0, q_len, kv_len;
    uint32_t rows, first;    // rows of the sequence, the tile's first
    uint32_t chunk, split;   // steps of a share, the item's share
    uint32_t splits;         // shares of the sequence's keys
    bool ok;
};

// Inclusive sum over the wave's lanes (row_shr 1, 2, 4, 8 and the rows' last
// lanes broadcast on).
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false);
    return v;
}

__device__ __forceinline__ uint32_t wave_total(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(v), kWave - 1);
}

__device__ __forceinline__ uint32_t att_steps(uint32_t keys) { return (keys + kAttStep - 1) / kAttStep; }

// Items are numbered through the sequences: a sequence has ceil(len * group /
// kRows) tiles of ceil(steps / chunk) shares each.  The chunk is the same for all
// sequences, so that items take equally long however ragged the lengths are: the
// least (to an eighth) with which there are no more than `target`.  The host
// knows no lengths; the grid has as many items as there can be, and those past
// the last are empty.
template <uint32_t kRows>
__device__ __forceinline__ AttItem att_item(const AttArgs& a, uint32_t item) {
    AttItem t = {};
    const uint32_t lim = (uint32_t)a.tokens;
    const uint32_t cap = a.c.num_pages ? a.max_pages << a.c.shift : 0;
    uint32_t q0 = 0, len = 0, kv = 0;
    auto read = [&](uint32_t s0) {
        const uint32_t s = s0 + lane_id();
        q0 = len = kv = 0;
        if (s < a.num_seqs) {
            q0 = min(a.starts[s], lim);
            const uint32_t q1 = min(a.starts[s + 1], lim);
            len = q1 > q0 ? q1 - q0 : 0;
            kv = min(a.lens[s], cap);
        }
    };
    auto tiles = [&] { return (len * a.group + kRows - 1) / kRows; };
    t.chunk = 0xffffffffu;
    if (a.target) {
        // Sum over the sequences of f(tiles, steps).
        const bool one = a.num_seqs <= kWave;
        if (one) read(0);
        auto sum = [&](auto f) {
            uint64_t all = 0;
            for (uint32_t s0 = 0; s0 < a.num_seqs; s0 += kWave) {
                if (!one) read(s0);
                all += f((uint64_t)tiles(), att_steps(kv));
            }
            const uint32_t lo = wave_total((uint32_t)all & 0xffffffu), hi = wave_total((uint32_t)(all >> 24));
            return ((uint64_t)hi << 24) + lo;
        };
        const uint64_t all = sum([](uint64_t n, uint32_t steps) { return n * steps; });
        uint64_t chunk = max((all + a.target - 1) / a.target, (uint64_t)kAttMinChunk);
        // a chunk of all steps leaves a share a tile
        while (chunk < kAttMaxSteps && sum([&](uint64_t n, uint32_t steps) {
                   return n * max((steps + (uint32_t)chunk - 1) / (uint32_t)chunk, 1u);
               }) > a.target)
            chunk += (chunk + 7) / 8;
        t.chunk = (uint32_t)min(chunk, (uint64_t)kAttMaxSteps);
    }
    uint32_t before = 0;  // items of the sequences gone by
    for (uint32_t s0 = 0; s0 < a.num_seqs; s0 += kWave) {
        if (!a.target || a.num_seqs > kWave) read(s0);  // else it has been
        const uint32_t splits = a.target ? max((att_steps(kv) + t.chunk - 1) / t.chunk, 1u) : 1u;
        const uint32_t count = tiles() * splits, sum = wave_scan(count);
        const uint32_t all = (uint32_t)__builtin_amdgcn_readlane((int)sum, kWave - 1);
        if (item - before >= all) {
            before += all;
            continue;
        }
        const int lane = (int)__popcll(__ballot(sum <= item - before));  // sequences that end before the item
        t.seq = s0 + lane;
        t.q0 = (uint32_t)__builtin_amdgcn_readlane((int)q0, lane);
        t.q_len = (uint32_t)__builtin_amdgcn_readlane((int)len, lane);
        t.kv_len = (uint32_t)__builtin_amdgcn_readlane((int)kv, lane);
        t.splits = (uint32_t)__builtin_amdgcn_readlane((int)splits, lane);
        const uint32_t n = (uint32_t)__builtin_amdgcn_readlane((int)count, lane);
        const uint32_t at = item - before - ((uint32_t)__builtin_amdgcn_readlane((int)sum, lane) - n);
        t.rows = t.q_len * a.group;
        t.split = at % t.splits;
        t.first = (n / t.splits - 1 - at / t.splits) * kRows;  // the rows that see the most keys first
        t.ok = true;
        return t;
    }
    return t;
}

// Keys that row r of the sequence sees: all, or those up to its own position,
// the last new token sitting at kv_len - 1.
__device__ __forceinline__ uint32_t att_limit(const AttArgs& a, const AttItem& t, uint32_t r) {
    if (!a.causal) return t.kv_len;
    const uint32_t after = t.q_len - 1 - r / a.group;
    return t.kv_len > after ? t.kv_len - after : 0;
}

__device__ __forceinline__ uint32_t perm(uint32_t hi, uint32_t lo, uint32_t sel) {
    return __builtin_amdgcn_perm(hi, lo, sel);
}

template <int kSel>
__device__ __forceinline__ uint32_t cvt2(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, kSel));
}

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
}

// Two floats as bf16 (to nearest) in one register, and what that left over.
__device__ __forceinline__ uint32_t pack_bf16(float x, float y, float* rx, float* ry) {
    const bf16x2 v = {(__bf16)x, (__bf16)y};
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    *rx = x - __uint_as_float(u << 16);
    *ry = y - __uint_as_float(u & 0xffff0000u);
    return u;
}

// Row r's query.
__device__ __forceinline__ const float* att_query(const AttArgs& a, const AttItem& t, uint32_t head, uint32_t r) {
    return a.q + (uint64_t)(t.q0 + r / a.group) * a.q_stride + (uint64_t)(head * a.group + r % a.group) * a.dim;
}

// What a lane loads of one 16-token tile.
template <int NB>
struct AttKV {
    static constexpr int kC = NB < 4 ? 1 : NB / 4;  // 16-byte pieces
    uint32_t k[NB];   // token n's codes of group g, eight dimensions a dword
    u32x4 v[kC];      // four tokens of chunk n (or n / 2, or 2n and 2n + 1)
    uint32_t ks[kC];  // K's scale bytes
    uint32_t vs;      // V's scale bytes of tokens 4g .. 4g + 3
    uint32_t valid;   // tokens of the tile that exist
};

// A value that the compiler takes as new, so that 32-bit offsets stay 32 bits wide
// beside their use (a load from a scalar base) and no 64-bit sums are kept.
__device__ __forceinline__ uint32_t opaque(uint32_t v) {
    asm("" : "+v"(v));
    return v;
}

// Adds v of the lanes N places round in each row of 16.
template <int N>
__device__ __forceinline__ float add_ror(float v) {
    return v + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x120 + N, 0xf, 0xf, true));
}

// NB: blocks of 32 dimensions that the tiles hold (2, 4 or 8), nb <= NB of them
// in use.  kSlot: query rows of a matrix tile's 16 columns.  16: a product for
// each of q's three terms and each of p's two.  With 8 or 4 rows (a decode step's
// query heads) the terms lie side by side in the columns instead, column = slot *
// kSlot + row: one product takes two or all three of q's terms and both of p's,
// and the slots' scores are added across lanes.
// R: 16-row tiles of a wave.  An item's rows are kSlot, or 64 R: its waves deal
// out the rows, and where there are too few rows for four waves, the tokens,
// whose parts they join at the end.
template <int NB, int R, int kSlot>
struct AttShape {
    static constexpr uint32_t kWaveRows = kSlot < 16 ? kSlot : 16 * R;
    static constexpr uint32_t kRows = kSlot < 16 ? kSlot : 16 * R * kAttWaves;
    static constexpr int kSide = 16 / kSlot;                      // terms side by side
    static constexpr int kQ = (kAttTerms + kSide - 1) / kSide;    // products for a score
    static constexpr int kP = kSlot == 16 ? 2 : 1;                // products for an output
};

template <int NB, int R, int kSlot, int kPerSimd>
__global__ __launch_bounds__(kAttBlock) __attribute__((amdgpu_waves_per_eu(kPerSimd, kPerSimd)))
void att_kernel(AttArgs a) {
    using Shape = AttShape<NB, R, kSlot>;
    constexpr uint32_t kRows = Shape::kRows, kWaveRows = Shape::kWaveRows;
    constexpr int kQ = Shape::kQ, kP = Shape::kP, kC = AttKV<NB>::kC;
    constexpr int kJ = 2 * NB;  // dimensions of a lane's part of a row, and O tiles
    const uint32_t lane = threadIdx.x % kWave, n = lane % 16, g = lane / 16;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave));
    // Key heads change fastest: workgroups go round the 8 XCDs, and every XCD gets
    // its part of the items, of which the last may be empty.
    const uint32_t head = blockIdx.x % a.c.kv_heads, item = a.item0 + blockIdx.x / a.c.kv_heads;
    const AttItem t = att_item<kRows>(a, item);
    if (!t.ok) return;
    const uint32_t nb = a.c.nb;
    // The waves' rows: one, two or four groups of them; the waves of a group share
    // its tokens.
    const uint32_t left = min(t.rows - t.first, kRows);
    const uint32_t groups = left <= kWaveRows ? 1 : left <= 2 * kWaveRows ? 2 : 4;
    const uint32_t share_of = kAttWaves / groups, part = wave / groups;
    const uint32_t r0 = t.first + (wave % groups) * kWaveRows;  // the wave's first row
    const uint32_t r1 = min(r0 + kWaveRows, t.rows);            // its end; r0 or less: no rows
    const uint32_t last_row = min(t.first + kRows, t.rows) - 1;

    // Tokens of this split, then of this wave.
    const uint32_t steps = att_steps(att_limit(a, t, last_row));
    const uint32_t lo = t.splits > 1 ? t.split * t.chunk : 0, hi = t.splits > 1 ? min(lo + t.chunk, steps) : steps;
    if (t.splits > 1 && lo >= hi) return;  // the joining kernel knows
    const uint32_t min_limit = att_limit(a, t, min(r0, t.rows - 1));
    const uint32_t end = r0 < r1 ? min(hi, att_steps(att_limit(a, t, r1 - 1))) : 0;

    uint32_t limit[R];
    u32x4 qf[R][kQ][NB];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const uint32_t row = r0 + 16 * r + n % kSlot, slot = n / kSlot;
        const bool live = row < r1;
        limit[r] = live ? att_limit(a, t, row) : 0;
        const float* qp = att_query(a, t, head, live ? row : 0);
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const uint32_t d0 = g * 8 * NB + 8 * j;
            float x[8];
            if (live && d0 + 8 <= a.dim) {
                const f32x4 u = (f32x4)*reinterpret_cast<const f32x4_a4*>(qp + d0);
                const f32x4 v = (f32x4)*reinterpret_cast<const f32x4_a4*>(qp + d0 + 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[i] = u[i];
                    x[4 + i] = v[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = live && d0 + i < a.dim ? qp[d0 + i] : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float u = x[2 * i] * a.scale_log2, v = x[2 * i + 1] * a.scale_log2;
                uint32_t term[kAttTerms];
#pragma unroll
                for (int k = 0; k < kAttTerms; ++k) {  // the top 16 bits, then what they leave
                    const uint32_t ub = __float_as_uint(u), vb = __float_as_uint(v);
                    term[k] = perm(vb, ub, 0x07060302u);
                    u -= __uint_as_float(ub & 0xffff0000u);
                    v -= __uint_as_float(vb & 0xffff0000u);
                }
#pragma unroll
                for (int k = 0; k < kQ; ++k) {
                    uint32_t w = 0;
#pragma unroll
                    for (int at = 0; at < Shape::kSide; ++at)
                        if (k * Shape::kSide + at < kAttTerms && slot == (uint32_t)at) w = term[k * Shape::kSide + at];
                    qf[r][k][j][i] = w;
                }
            }
        }
    }

    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    const float ninf = -__builtin_inff();
    f32x4 o[R][kJ];
    float m[R], l[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        m[r] = ninf;
        l[r] = 0.0f;
#pragma unroll
        for (int j = 0; j < kJ; ++j) o[r][j] = zero;
    }

    // Loads have no conditions on their way, so that a step's can be waited for
    // while the next one's are in flight: a tile past the end is one of page 0 with
    // no tokens, blocks past nb are read from the last one (q is zero there, and
    // what they add to the output is not stored).
    typedef const __attribute__((address_space(4))) uint32_t* ScalarPtr;
    const ScalarPtr table = (ScalarPtr)(uintptr_t)(a.table + (uint64_t)t.seq * a.max_pages);
    const uint32_t last_page = t.kv_len ? (t.kv_len - 1) >> a.c.shift : 0;
    auto page_of = [&](uint32_t tt) { return table[min(tt * 16 >> a.c.shift, last_page)]; };
    const uint32_t stride = share_of;
    uint32_t koff[kC], ksoff[kC], voff[kC], vsoff = 0;
#pragma unroll
    for (int c = 0; c < kC; ++c) {
        const uint32_t np = a.c.page * nb, kb = min(NB == 2 ? g / 2 : g * kC + c, nb - 1);
        koff[c] = n * nb * 16 + kb * 16 + (NB == 2 ? g % 2 * 8 : 0);
        ksoff[c] = np * 32 + n * nb + kb;
        const uint32_t chunk = min(NB == 2 ? n / 2 : n * kC + c, 4 * nb - 1);
        voff[c] = np * 16 + (g * 4 * nb + chunk) * 16;
        if (c == 0) vsoff = np * 33 + chunk / 4 * 16 + 4 * g;
    }
    auto load = [&](uint32_t tt, uint32_t page, AttKV<NB>& x) {
        x.valid = min(t.kv_len - min(t.kv_len, tt * 16), 16u);
        if (page >= a.c.num_pages) page = 0, x.valid = 0;  // a page that does not exist has no tokens
        const uint32_t t0 = (tt * 16) & (a.c.page - 1);
        const uint8_t* base = a.cache + (uint64_t)page * a.c.page_bytes + (uint64_t)head * a.c.head_bytes;
        const uint8_t* codes = base + t0 * nb * 16;
        const uint8_t* scales = base + t0 * nb;
#pragma unroll
        for (int c = 0; c < kC; ++c) {
            if constexpr (NB == 2) {
                const u32x2 u = *reinterpret_cast<const u32x2*>(codes + opaque(koff[c]));
                x.k[0] = u.x;
                x.k[1] = u.y;
            } else {
                const u32x4 u = *reinterpret_cast<const u32x4*>(codes + opaque(koff[c]));
#pragma unroll
                for (int i = 0; i < 4; ++i) x.k[4 * c + i] = u[i];
            }
            x.v[c] = *reinterpret_cast<const u32x4*>(codes + opaque(voff[c]));
            x.ks[c] = scales[opaque(ksoff[c])];
        }
        x.vs = *reinterpret_cast<const uint32_t*>(scales + opaque(vsoff));
    };

    auto work = [&](uint32_t step, AttKV<NB> (&cur)[2], uint32_t page0, uint32_t page1) {
        // Scores: tokens 4g + i of both tiles, in powers of two.
        f32x4 s[R][2];
#pragma unroll
        for (int r = 0; r < R; ++r) s[r][0] = s[r][1] = zero;
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const float sc = __uint_as_float(cur[x].ks[j / 4] << 23);
                const uint32_t code = cur[x].k[j];
                const u32x4 kf = {cvt2<0>(code, sc), cvt2<1>(code, sc), cvt2<2>(code, sc), cvt2<3>(code, sc)};
#pragma unroll
                for (int k = kQ - 1; k >= 0; --k)
#pragma unroll
                    for (int r = 0; r < R; ++r) s[r][x] = mfma(kf, qf[r][k][j], s[r][x]);
            }
        if constexpr (kSlot < 16) {
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[0][x][i] = add_ror<8>(s[0][x][i]);
                    if constexpr (kSlot == 4) s[0][x][i] = add_ror<4>(s[0][x][i]);
                }
        }
        const uint32_t at = step * kAttStep;
        // Every row of the wave sees every token of the step: no masks.
        const bool whole = at + kAttStep <= min_limit && cur[0].valid + cur[1].valid == kAttStep;
        bool nan_v = false;
        if (!whole) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const uint32_t have_x = at + 16 * x + cur[x].valid;  // the tile's tokens end here
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (at + 16 * x + 4 * g + i >= min(limit[r], have_x)) s[r][x][i] = ninf;
                uint32_t vs = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t b = cur[x].vs >> 8 * i & 0xffu;
                    if (4 * g + i >= cur[x].valid) b = 127;
                    if (b == kQ4NanScale) nan_v = true, b = 127;
                    vs |= b << 8 * i;
                }
                cur[x].vs = vs;
            }
        }
        // Running maximum, probabilities and their sum; bf16 terms.
        u32x4 pf[R][kP];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float mx = fmaxf(fmaxf(fmaxf(s[r][0][0], s[r][0][1]), fmaxf(s[r][0][2], s[r][0][3])),
                             fmaxf(fmaxf(s[r][1][0], s[r][1][1]), fmaxf(s[r][1][2], s[r][1][3])));
            if (__any(mx > m[r])) {
                mx = fmaxf(mx, __shfl_xor(mx, 16, kWave));
                mx = fmaxf(mx, __shfl_xor(mx, 32, kWave));
                const float mn = fmaxf(m[r], mx);
                const float f = mn > m[r] ? __builtin_amdgcn_exp2f(m[r] - mn) : 1.0f;
                m[r] = mn;
                l[r] *= f;
#pragma unroll
                for (int j = 0; j < kJ; ++j) o[r][j] *= f;
            }
            const float base = m[r] == ninf ? 0.0f : m[r];
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    float p0 = __builtin_amdgcn_exp2f(s[r][x][i] - base);
                    float p1 = __builtin_amdgcn_exp2f(s[r][x][i + 1] - base);
                    l[r] += p0 + p1;
                    float e0, e1, u0, u1;
                    const uint32_t top = pack_bf16(p0, p1, &e0, &e1);
                    if constexpr (kSlot == 16) {
                        pf[r][0][2 * x + i / 2] = top;
                        pf[r][1][2 * x + i / 2] = pack_bf16(e0, e1, &u0, &u1);
                    } else {  // slot 0 holds the first term, slot 1 the second; the others are not read
                        pf[r][0][2 * x + i / 2] = n < kSlot ? top : pack_bf16(e0, e1, &u0, &u1);
                    }
                }
        }
        // V: four dwords a tile are four tokens x eight dimensions; an operand is
        // eight tokens of one dimension.
        float vsc[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) vsc[i] = __uint_as_float((cur[i >> 2].vs >> 8 * (i & 3) & 0xffu) << 23);
#pragma unroll
        for (int p = 0; p < NB; ++p) {  // pair of dimensions 2p, 2p + 1
            uint32_t v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                uint32_t code = cur[i >> 2].v[NB == 8 ? p >> 2 : 0][i & 3];
                if (NB == 2) code >>= (n & 1) * 16;  // the lane's four dimensions of the chunk
                v[i] = (p & 3) == 0   ? cvt2<0>(code, vsc[i])
                       : (p & 3) == 1 ? cvt2<1>(code, vsc[i])
                       : (p & 3) == 2 ? cvt2<2>(code, vsc[i])
                                      : cvt2<3>(code, vsc[i]);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                u32x4 vf;
#pragma unroll
                for (int i = 0; i < 4; ++i) vf[i] = perm(v[2 * i + 1], v[2 * i], h ? 0x07060302u : 0x05040100u);
#pragma unroll
                for (int k = kP - 1; k >= 0; --k)
#pragma unroll
                    for (int r = 0; r < R; ++r) o[r][2 * p + h] = mfma(vf, pf[r][k], o[r][2 * p + h]);
            }
        }
        // A NaN block of a token that some rows do not see: its 32 dimensions of
        // the rows that do.
        if (!whole && __any(nan_v)) {
            for (uint32_t x = 0; x < 2; ++x) {
                const uint32_t page = x ? page1 : page0, t0 = (at + 16 * x) & (a.c.page - 1);
                const uint32_t valid = x ? cur[1].valid : cur[0].valid;
                const uint8_t* base = a.cache + (uint64_t)page * a.c.page_bytes + (uint64_t)head * a.c.head_bytes;
                for (uint32_t b = 0; b < nb; ++b)
                    for (uint32_t i = 0; i < valid; ++i)
                        if (base[q4_v_scale(a.c, t0 + i, b)] == kQ4NanScale)
#pragma unroll
                            for (int r = 0; r < R; ++r)
                                if (at + 16 * x + i < limit[r])
#pragma unroll
                                    for (int k = 0; k < 4; ++k)
                                        if ((NB * (4 * g + k)) / 16 == b)
#pragma unroll
                                            for (int j = 0; j < kJ; ++j) o[r][j][k] = __uint_as_float(0x7fc00000u);
            }
        }
    };

    // Two steps in turn: one's loads are in flight while the other is worked on,
    // the pages of the one after that on their way.
    uint32_t step = lo + part;
    if (step < end) {
        AttKV<NB> kv[2][2];
        uint32_t pg[2][2], ahead[2];
        auto fetch = [&](uint32_t st, int to) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                pg[to][x] = ahead[x];
                load(2 * st + x, ahead[x], kv[to][x]);
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) ahead[x] = page_of(2 * (st + stride) + x);
        };
        ahead[0] = page_of(2 * step);
        ahead[1] = page_of(2 * step + 1);
        fetch(step, 0);
        for (;;) {
            fetch(step + stride, 1);
            work(step, kv[0], pg[0][0], pg[0][1]);
            step += stride;
            if (step >= end) break;
            fetch(step + stride, 0);
            work(step, kv[1], pg[1][0], pg[1][1]);
            step += stride;
            if (step >= end) break;
        }
    }

#pragma unroll
    for (int r = 0; r < R; ++r) {
        l[r] += __shfl_xor(l[r], 16, kWave);
        l[r] += __shfl_xor(l[r], 32, kWave);
    }
    // Lane (n, g) has dimensions kJ (4g + i) + j of row n in o[.][j][i].
    const uint64_t part0 = ((uint64_t)item * a.c.kv_heads + head) * kRows;
    const uint32_t dp = 32 * nb;
    float* const pm = a.part;  // [rows][2] of all, then [rows][dp] of all
    float* const po = a.part + (uint64_t)a.items * a.c.kv_heads * kRows * 2;
    // `count` values from dimension d of the sequence's row rr, not yet divided.
    auto store_row = [&](uint32_t rr, float mm, float ll, uint32_t d, const float* v, auto count) {
        constexpr int kCount = decltype(count)::value;
        if (t.splits > 1) {
            const uint64_t at = part0 + (rr - t.first);
            if (d == 0) {
                pm[at * 2] = mm;
                pm[at * 2 + 1] = ll;
            }
            float* p = po + at * dp + d;
#pragma unroll
            for (int i = 0; i < kCount; i += 4)
                if (d + i < dp) *reinterpret_cast<f32x4*>(p + i) = {v[i], v[i + 1], v[i + 2], v[i + 3]};
        } else {
            const float f = ll == 0.0f ? 0.0f : 1.0f / ll;
            float* p = a.out + ((uint64_t)(t.q0 + rr / a.group) * a.q_heads + head * a.group + rr % a.group) * a.dim + d;
#pragma unroll
            for (int i = 0; i < kCount; i += 4) {
                float u[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) u[k] = ll == 0.0f ? 0.0f : v[i + k] * f;
                if (d + i + 4 <= a.dim) {
                    *reinterpret_cast<f32x4_a4*>(p + i) = {u[0], u[1], u[2], u[3]};
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (d + i + k < a.dim) p[i + k] = u[k];
                }
            }
        }
    };
    if (groups == kAttWaves) {
        if constexpr (kSlot == 16) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const uint32_t row = r0 + 16 * r + n;
                if (row >= r1) continue;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float v[kJ];
#pragma unroll
                    for (int j = 0; j < kJ; ++j) v[j] = o[r][j][i];
                    store_row(row, m[r], l[r], kJ * (4 * g + i), v, std::integral_constant<int, kJ>());
                }
            }
        }
        return;
    }
    // Join the waves of a group: to the common maximum, then add (and the second
    // term's column to the first's).
    constexpr int kPitch = 16 * kJ + 4;
    __shared__ float sm[kAttWaves][16], sl[kAttWaves][16];
    __shared__ __attribute__((aligned(16))) float so[kAttWaves][16][kPitch];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        __syncthreads();
        if (g == 0) {
            sm[wave][n] = m[r];
            sl[wave][n] = l[r];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < kJ; j += 4)
                *reinterpret_cast<f32x4*>(&so[wave][n][kJ * (4 * g + i) + j]) = {o[r][j][i], o[r][j + 1][i],
                                                                                o[r][j + 2][i], o[r][j + 3][i]};
        __syncthreads();
        constexpr uint32_t kTall = kSlot < 16 ? kSlot : 16;  // rows of one group's tile
        constexpr uint32_t kQuads = 4 * kJ;                  // float4 of a row
        for (uint32_t i = threadIdx.x; i < groups * kTall * kQuads; i += kAttBlock) {
            const uint32_t d = i % kQuads * 4, row = i / kQuads % kTall, gr = i / kQuads / kTall;
            const uint32_t rr = t.first + gr * kWaveRows + 16 * r + row;
            if (rr >= t.rows) continue;
            float mm = ninf, ll = 0.0f;
            for (uint32_t w = gr; w < kAttWaves; w += groups) mm = fmaxf(mm, sm[w][row]);
            float v[4] = {0.f, 0.f, 0.f, 0.f};
            for (uint32_t w = gr; w < kAttWaves; w += groups) {
                // a wave that saw nothing holds zeros (or NaN, which stays)
                const float f = sm[w][row] == ninf ? 1.0f : __builtin_amdgcn_exp2f(sm[w][row] - mm);
                ll += sl[w][row] * f;
                f32x4 u = *reinterpret_cast<const f32x4*>(&so[w][row][d]);
                if (kSlot < 16) u += *reinterpret_cast<const f32x4*>(&so[w][row + kSlot % 16][d]);
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] += u[k] * f;
            }
            store_row(rr, mm, ll, d, v, std::integral_constant<int, 4>());
        }
    }
}

// Joins the shares of a tile, kJoinRows rows at a time: their maxima and sums
// through LDS, then a thread has four dimensions of a row and every kth share.
constexpr uint32_t kJoinRows = 4;

template <uint32_t kRows>
__global__ __launch_bounds__(kAttJoin) void att_join_kernel(AttArgs a) {
    __shared__ float2 ml[kJoinRows][kAttMaxSplits];
    __shared__ f32x4 red[kAttJoin];
    const uint32_t head = blockIdx.x % a.c.kv_heads, item = a.item0 + blockIdx.x / a.c.kv_heads;
    const AttItem t = att_item<kRows>(a, item);
    if (!t.ok || t.split || t.splits == 1) return;
    const uint32_t last_row = min(t.first + kRows, t.rows) - 1;
    const uint32_t used = (att_steps(att_limit(a, t, last_row)) + t.chunk - 1) / t.chunk;
    const uint64_t next = (uint64_t)a.c.kv_heads * kRows;  // rows to the next share's
    const float* po = a.part + (uint64_t)a.items * a.c.kv_heads * kRows * 2;
    const uint32_t dp = 32 * a.c.nb, quads = dp / 4, group = kJoinRows * quads, groups = kAttJoin / group;
    const uint32_t gr = threadIdx.x / group, row = threadIdx.x % group / quads, d = threadIdx.x % quads * 4;
    for (uint32_t row0 = 0; row0 < kRows && t.first + row0 < t.rows; row0 += kJoinRows) {
        const uint64_t part0 = ((uint64_t)item * a.c.kv_heads + head) * kRows + row0;
        const float2* pm = reinterpret_cast<const float2*>(a.part) + part0;
        __syncthreads();
        // rows past the sequence's hold anything and are not stored
        for (uint32_t i = threadIdx.x; i < used * kJoinRows; i += kAttJoin)
            ml[i % kJoinRows][i / kJoinRows] = pm[i / kJoinRows * next + i % kJoinRows];
        __syncthreads();
        const float ninf = -__builtin_inff();
        float mm = ninf, ll = 0.0f;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        if (gr < groups) {
            for (uint32_t z = 0; z < used; ++z) mm = fmaxf(mm, ml[row][z].x);
            const float* p = po + (part0 + row) * dp + d;
#pragma unroll 8
            for (uint32_t z = gr; z < used; z += groups) {
                const float2 u = ml[row][z];
                // a share that saw nothing holds zeros (or NaN, which stays)
                const float f = u.x == ninf ? 1.0f : __builtin_amdgcn_exp2f(u.x - mm);
                v += *reinterpret_cast<const f32x4*>(p + z * next * dp) * f;
            }
        }
        red[threadIdx.x] = v;
        __syncthreads();
        const uint32_t rr = t.first + row0 + row;
        if (gr == 0 && rr < t.rows) {
            for (uint32_t k = 1; k < groups; ++k) v += red[threadIdx.x + k * group];
            for (uint32_t z = 0; z < used; ++z) {
                const float2 u = ml[row][z];
                ll += u.x == ninf ? u.y : u.y * __builtin_amdgcn_exp2f(u.x - mm);
            }
            float* out = a.out + ((uint64_t)(t.q0 + rr / a.group) * a.q_heads + head * a.group + rr % a.group) * a.dim;
            const float f = 1.0f / ll;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (d + k < a.dim) out[d + k] = ll == 0.0f ? 0.0f : v[k] * f;
        }
    }
}

// Rows of an item: a decode step's query heads in a few columns, or rows for four
// waves.
struct AttPlan {
    int slot, r;    // kSlot, R
    uint32_t rows;  // kRows
    uint32_t items, target;
    uint64_t bytes;  // workspace
};

static int att_plan(uint64_t num_seqs, uint64_t tokens, uint64_t q_heads, uint64_t kv_heads, uint64_t page_size,
                    uint64_t max_pages, uint32_t nb, AttPlan* p) {
    const uint64_t group = q_heads / kv_heads, rows = tokens * group;
    p->slot = rows <= 4 * num_seqs ? 4 : rows <= 8 * num_seqs ? 8 : 16;
    p->r = p->slot < 16 || nb > 4 ? 1 : 2;
    p->rows = p->slot < 16 ? p->slot : 64u * p->r;
    const uint64_t tiles = rows / p->rows + num_seqs;
    if (tiles > 0x3fffffull) return KORE_HIP_ERR_OVERFLOW;
    // Workgroups that the keys are cut for: what the chip holds at once.
    const uint64_t want = p->slot == 4 && nb <= 4 ? 768 : 512;
    const uint64_t busy = std::max(std::min(num_seqs, tokens), rows / p->rows) * kv_heads;
    const uint64_t shares = max_pages * page_size / (kAttMinChunk * kAttStep);  // of the longest sequence
    const bool cut = busy < (p->slot < 16 ? 2 * want : want / 2) && shares > 1;
    p->target = cut ? (uint32_t)std::min<uint64_t>({(want + kv_heads - 1) / kv_heads, tiles * shares, kAttMaxSplits}) : 0;
    p->items = std::max((uint32_t)tiles, p->target);
    p->bytes = cut ? (uint64_t)p->items * kv_heads * p->rows * (2 + 32ull * nb) * 4 : 0;
    return KORE_HIP_OK;
}

static int att_check(uint64_t num_seqs, uint64_t tokens, uint64_t q_heads, uint64_t kv_heads, uint64_t head_dim,
                     uint64_t num_pages, uint64_t page_size, uint64_t max_pages, Q4Cache* c, AttPlan* p,
                     uint64_t* bytes) {
    const int st = q4_layout(num_pages, page_size, kv_heads, head_dim, c, bytes);
    if (st != KORE_HIP_OK) return st;
    if (kv_heads == 0 || q_heads % kv_heads) return KORE_HIP_ERR_BAD_DIM;
    if (num_seqs > 0x7fffffffull || tokens > 0x7fffffffull || q_heads > 65535u ||
        max_pages > 0x7fffffffull / page_size || (num_seqs && max_pages > kMaxElements / num_seqs) ||
        tokens * q_heads > 0xffffffffull)
        return KORE_HIP_ERR_OVERFLOW;
    return att_plan(num_seqs, tokens, q_heads, kv_heads, page_size, max_pages, c->nb, p);
}

template <int NB, int R, int kSlot, int kPerSimd>
static void att_launch_shape(const AttArgs& a, bool join, dim3 grid, hipStream_t s) {
    if (join)
        hipLaunchKernelGGL((att_join_kernel<AttShape<NB, R, kSlot>::kRows>), grid, dim3(kAttJoin), 0, s, a);
    else
        hipLaunchKernelGGL((att_kernel<NB, R, kSlot, kPerSimd>), grid, dim3(kAttBlock), 0, s, a);
}

static void att_launch(const AttArgs& a, const AttPlan& p, bool join, dim3 grid, hipStream_t s) {
    const int nb = a.c.nb <= 2 ? 2 : a.c.nb <= 4 ? 4 : 8;
    auto any = [&](auto blocks) {
        constexpr int NB = decltype(blocks)::value;
        if (p.slot == 4) att_launch_shape<NB, 1, 4, NB == 8 ? 2 : 3>(a, join, grid, s);
        else if (p.slot == 8) att_launch_shape<NB, 1, 8, NB == 8 ? 1 : 2>(a, join, grid, s);
        else att_launch_shape<NB, NB == 8 ? 1 : 2, 16, NB == 8 ? 1 : 2>(a, join, grid, s);
    };
    if (nb == 2) any(std::integral_constant<int, 2>());
    else if (nb == 4) any(std::integral_constant<int, 4>());
    else any(std::integral_constant<int, 8>());
}

static bool att_overlap(const void* a, uint64_t na, const void* b, uint64_t nb) {
    const char *p = (const char*)a, *q = (const char*)b;
    return p < q + nb && q < p + na;
}

}  // namespace kore

using namespace kore;

extern "C" uint64_t kore_hip_attention_q4_workspace_bytes(uint64_t num_seqs, uint64_t tokens, uint64_t q_heads,
                                                          uint64_t kv_heads, uint64_t head_dim, uint64_t page_size,
                                                          uint64_t max_pages) {
    if (num_seqs == 0 || tokens == 0 || q_heads == 0) return 0;
    Q4Cache c;
    AttPlan p;
    uint64_t bytes;
    if (att_check(num_seqs, tokens, q_heads, kv_heads, head_dim, 0, page_size, max_pages, &c, &p, &bytes)) return 0;
    return p.bytes;
}

extern "C" int kore_hip_attention_q4_f32(const float* q, const uint8_t* cache, const uint32_t* page_table,
                                         const uint32_t* kv_lens, const uint32_t* q_starts, float* out,
                                         float* workspace, uint64_t workspace_bytes, uint64_t num_seqs,
                                         uint64_t tokens, uint64_t q_heads, uint64_t kv_heads, uint64_t head_dim,
                                         uint64_t num_pages, uint64_t page_size, uint64_t max_pages,
                                         uint64_t q_stride, float scale, int causal, kore_stream_t stream) {
    if (num_seqs == 0 || tokens == 0 || q_heads == 0 || head_dim == 0) return KORE_HIP_OK;
    AttArgs a = {};
    AttPlan p;
    uint64_t bytes, span;
    const int st = att_check(num_seqs, tokens, q_heads, kv_heads, head_dim, num_pages, page_size, max_pages, &a.c, &p,
                             &bytes);
    if (st != KORE_HIP_OK) return st;
    const uint64_t row = q_heads * head_dim;
    a.q_stride = q_stride ? q_stride : row;
    if (a.q_stride < row) return KORE_HIP_ERR_BAD_DIM;
    if (!mul_ok(tokens, a.q_stride, &span) || span > kMaxElements) return KORE_HIP_ERR_OVERFLOW;
    if (!q || !kv_lens || !q_starts || !out || (max_pages && !page_table) || (num_pages && !cache) ||
        (p.bytes && !workspace))
        return KORE_HIP_ERR_NULL_PTR;
    if ((num_pages && !aligned16(cache)) || (p.bytes && (workspace_bytes < p.bytes || !aligned16(workspace))))
        return KORE_HIP_ERR_BAD_DIM;
    const uint64_t out_bytes = tokens * row * 4;
    if (att_overlap(out, out_bytes, q, ((tokens - 1) * a.q_stride + row) * 4) ||
        att_overlap(out, out_bytes, cache, bytes) || att_overlap(out, out_bytes, workspace, p.bytes) ||
        att_overlap(out, out_bytes, page_table, num_seqs * max_pages * 4) ||
        att_overlap(out, out_bytes, kv_lens, num_seqs * 4) || att_overlap(out, out_bytes, q_starts, num_seqs * 4 + 4))
        return KORE_HIP_ERR_ALIAS;
    a.q = q;
    a.cache = cache;
    a.table = page_table;
    a.lens = kv_lens;
    a.starts = q_starts;
    a.out = out;
    a.part = workspace;
    a.tokens = tokens;
    a.num_seqs = (uint32_t)num_seqs;
    a.q_heads = (uint32_t)q_heads;
    a.group = (uint32_t)(q_heads / kv_heads);
    a.max_pages = (uint32_t)max_pages;
    a.dim = (uint32_t)head_dim;
    a.items = p.items;
    a.target = p.target;
    a.scale_log2 = (float)((double)scale * 1.4426950408889634);
    a.causal = causal != 0;
    // A launch holds fewer than 2^32 threads: items in bands.
    const uint32_t band = (uint32_t)std::max<uint64_t>(1, 0x400000u / kv_heads);
    for (int join = 0; join < (p.target ? 2 : 1); ++join) {
        for (a.item0 = 0; a.item0 < p.items; a.item0 += band) {
            const uint32_t x = std::min(band, p.items - a.item0) * (uint32_t)kv_heads;
            att_launch(a, p, join != 0, dim3(x), (hipStream_t)stream);
            const int rc = launch_status();
            if (rc != KORE_HIP_OK) return rc;
        }
    }
    return KORE_HIP_OK;
}
