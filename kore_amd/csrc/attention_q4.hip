// attention_q4.hip -- softmax(scale q k^T) v over the paged 4-bit cache, for
// ragged sequences with any number of new tokens each.
//
// One pass over the keys with the running maximum and sum of the softmax; no
// scores in memory.  The rows of one key head are its query heads times the
// sequence's new tokens: row r = token * group + head.
//
// Arithmetic.  A cached value is a code times a power of two, exact in bf16, and
// gfx950 makes two of them with their scale in one instruction, so the matrix
// cores' bf16 form loses nothing on the cache's side.  A query value (times scale
// * log2 e, one f32 rounding) is cut into three bf16 terms of 8 bits each, which
// is all of its 24: every product q * k is exact and sums are f32.  Probabilities
// are cut the same way.  With two terms each (2^-18 of a probability lost) results
// were off by 2.4e-6 of themselves where f32 products are by 6e-7; the third costs
// a decode step nothing and a prompt a sixth more products.
// (The block-scaled product takes K's codes and scales as they lie, and q as six
// E4M3 terms; but its sum keeps only some 2^-19 of the largest product, so blocks
// of very different scales would cost accuracy that f32 has.)
//
// Both products are taken transposed, S^T = K Q^T and O^T = V^T P^T, so that a
// lane's scores, probabilities and outputs all belong to one row, its column:
// maximum, sum and rescaling are its own, but for a maximum over the four lane
// groups.  The operand P^T wants eight tokens of a row from each lane group; V's
// operand is taken for those eight that the lane has from S^T, so P moves between
// no lanes and through no memory.
//
// A masked token's score is -inf whatever its codes say.  Its V is finite (the
// scale of a token past the cache's length counts as 1); where V of a token
// that only later rows see is NaN, the product uses 1 for the scale and the
// rows that see it are set to NaN one by one.
//
// Bound and measured (MI355X; a copy of 2 GiB moves 4.5 TB/s, one that the last cache
// holds 8.2; a bf16 matrix product reaches 1402 TFLOP/s):
//   decode, HBM: 2 sequences of 131072 and 70320 tokens, 8 key heads of 128, 219 MB:
//     45.5 us (4.8 TB/s) and 7.0 to join; 45 of 8192 .. 2048, 256 MB: 60 and 5.4.
//     The conversion and softmax of a step, some 185 vector instructions, are issued
//     in 70 % of the cycles beside the loads.
//   one sequence of 2048 tokens: 7.6 + 4.2 us, two launches and their chains of loads.
//   prompt, matrix cores: 4096 tokens, 32 + 8 heads of 128, 137 GFLOP of which each is
//     three in bf16: 306 .. 327 us by the card, 1350 .. 1260 TFLOP/s in bf16 (matrix
//     cores busy in 60 % of the cycles, vector issue in 65 %).
//   chunks of 1023 and fewer after 2777 and fewer, 16 heads of 64: 98 us, a third of
//     it matrix cores: at 64 dimensions a step of a wave has 180 vector instructions
//     for 24 products, and their issue bounds it (68 % of all cycles).
#include <algorithm>
#include <type_traits>

#include "q4.hpp"

namespace kore {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kAttBlock = 256;
constexpr int kAttWaves = kAttBlock / kWave;
constexpr uint32_t kAttStep = 32;             // tokens of a step
constexpr uint32_t kAttMinChunk = 8;          // steps of a share, at least: two for each wave
constexpr uint32_t kAttMaxSteps = 1u << 27;   // more than 2^31 keys have
constexpr int kAttTerms = 3;                  // bf16 terms of a float
constexpr uint32_t kAttMaxSplits = 1024;
constexpr uint32_t kAttCus = 256;

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
    int search;             // many sequences: numbered with gaps, so that one can be found
    float scale_log2;
    int causal;
    Q4Cache c;
};

// A work item: kRows consecutive rows of one sequence and one share of its keys.
struct AttItem {
    uint32_t seq, q0, q_len, kv_len;
    uint32_t rows, first;    // rows of the sequence, the tile's first
    uint32_t chunk, split;   // steps of a share, the item's share
    uint32_t item;           // its number
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
// least (to an eighth; for more sequences than a wave's lanes hold, to a half) with
// which there are no more than `target`.  The host knows no lengths; the grid has as
// many items as there can be, and those past the last are empty.  kTiles: `number` is
// that of a tile, and its first item is meant.
template <uint32_t kRows, bool kTiles>
__device__ __forceinline__ AttItem att_item(const AttArgs& a, uint32_t number) {
    constexpr int kHeld = 4;  // sequences that a lane holds
    AttItem t = {};
    const uint32_t lim = (uint32_t)a.tokens;
    const uint32_t cap = a.c.num_pages ? a.max_pages << a.c.shift : 0;
    uint32_t q0[kHeld], len[kHeld], kv[kHeld];
    auto read = [&](uint32_t s0) {
#pragma unroll
        for (int k = 0; k < kHeld; ++k) {
            q0[k] = len[k] = kv[k] = 0;
            const uint32_t s = s0 + k * kWave + lane_id();
            if (k && s0 + k * kWave >= a.num_seqs) continue;
            const uint32_t from = a.starts[min(s, a.num_seqs)], to = a.starts[min(s + 1, a.num_seqs)];
            q0[k] = min(from, lim);
            len[k] = max(min(to, lim), q0[k]) - q0[k];
            kv[k] = min(a.lens[min(s, a.num_seqs - 1)], cap);
        }
    };
    auto tiles = [&](int k) { return (len[k] * a.group + kRows - 1) / kRows; };
    if (!kTiles && a.search) {
        // Sequence s begins at number floor(starts[s] * group / kRows) + s, which leaves
        // each as many numbers as it has tiles or more: found 64 sequences at a time.
        auto begin = [&](uint32_t s) { return min(a.starts[s], lim) * a.group / kRows + s; };
        uint32_t lo = 0;
        for (uint32_t n = a.num_seqs; n;) {
            const uint32_t each = (n + kWave - 1) / kWave, at = lane_id() * each;
            const uint32_t below = (uint32_t)__popcll(__ballot(at < n && begin(lo + min(at, n - 1)) <= number));
            if (below == 0) return t;  // before the first
            lo += (below - 1) * each;
            n = each == 1 ? 0 : min(each, n - (below - 1) * each);
        }
        t.q0 = min(a.starts[lo], lim);
        t.q_len = max(min(a.starts[lo + 1], lim), t.q0) - t.q0;
        t.kv_len = min(a.lens[lo], cap);
        t.rows = t.q_len * a.group;
        t.seq = lo;
        t.splits = 1;
        t.item = number;
        const uint32_t tile = number - begin(lo), n = (t.rows + kRows - 1) / kRows;
        t.ok = tile < n;
        t.first = t.ok ? (n - 1 - tile) * kRows : 0;
        return t;
    }
    const bool one = a.num_seqs <= kHeld * kWave;
    if (one) read(0);
    t.chunk = kAttMaxSteps;  // a share a tile
    if (a.target) {
        uint64_t all = 0;    // tiles times their steps
        uint32_t count = 0;  // tiles
        for (uint32_t s0 = 0; s0 < a.num_seqs; s0 += kHeld * kWave) {
            if (!one) read(s0);
            uint64_t n = 0;
            uint32_t m = 0;
#pragma unroll
            for (int k = 0; k < kHeld; ++k) {
                n += (uint64_t)tiles(k) * att_steps(kv[k]);
                m += tiles(k);
            }
            all += ((uint64_t)wave_total((uint32_t)(n >> 24)) << 24) + wave_total((uint32_t)n & 0xffffffu);
            count += wave_total(m);
        }
        // n tiles in shares of c steps make fewer than all / c + n: the chunk lies
        // between all / target and all / (target - n).
        if (count < a.target) {
            const uint64_t most = (all + a.target - count - 1) / (a.target - count);
            // at least: a 32nd of the average keys, from 8 steps to 32
            const uint64_t least = kAttMinChunk * (all >= 1024ull * count ? 4 : all >= 512ull * count ? 2 : 1);
            uint64_t chunk = max(one ? (all + a.target - 1) / a.target : most, least);
            while (chunk < most) {  // the sequences are in registers
                uint64_t n = 0;     // shares
#pragma unroll
                for (int k = 0; k < kHeld; ++k)
                    if (k == 0 || k * kWave < (int)a.num_seqs)
                        n += (uint64_t)tiles(k) * max((att_steps(kv[k]) + (uint32_t)chunk - 1) / (uint32_t)chunk, 1u);
                if (wave_total((uint32_t)min(n, (uint64_t)1 << 25)) <= a.target) break;
                chunk += (chunk + 7) / 8;
            }
            t.chunk = (uint32_t)min(chunk, (uint64_t)kAttMaxSteps);
        }
    }
    uint32_t before = 0, items = 0;  // numbers, items of the sequences gone by
    // Sequences of several tiles first: a prompt's chunk behind decode steps would
    // begin when they end (512 tokens behind 63 steps: 167 -> 129 us).
    const bool sorted = kRows > 8 && one;
    for (int few = 0; few < (sorted ? 2 : 1); ++few) {
        for (uint32_t s0 = 0; s0 < a.num_seqs; s0 += kHeld * kWave) {
            if (!one) read(s0);
#pragma unroll
            for (int k = 0; k < kHeld; ++k) {
                if (k && s0 + k * kWave >= a.num_seqs) break;
                const uint32_t splits = max((att_steps(kv[k]) + t.chunk - 1) / t.chunk, 1u);
                const uint32_t n = sorted && (tiles(k) > 1) == (few == 1) ? 0 : tiles(k);
                const uint32_t count = kTiles ? n : n * splits, sum = wave_scan(count);
                const uint32_t sum_items = kTiles ? wave_scan(n * splits) : sum;
                const uint32_t all = (uint32_t)__builtin_amdgcn_readlane((int)sum, kWave - 1);
                if (number - before >= all) {
                    before += all;
                    items += (uint32_t)__builtin_amdgcn_readlane((int)sum_items, kWave - 1);
                    continue;
                }
                // sequences that end before it
                const int lane = (int)__popcll(__ballot(sum <= number - before));
                auto of = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); };
                t.seq = s0 + k * kWave + lane;
                t.q0 = of(q0[k]);
                t.q_len = of(len[k]);
                t.kv_len = of(kv[k]);
                t.splits = of(splits);
                const uint32_t mine = of(n), at = number - before - (of(sum) - of(count));
                const uint32_t tile = kTiles ? at : at / t.splits;
                t.split = kTiles ? 0 : at % t.splits;
                t.item = kTiles ? items + of(sum_items) - (mine - tile) * t.splits : number;
                t.rows = t.q_len * a.group;
                t.first = (mine - 1 - tile) * kRows;  // the rows that see the most keys first
                t.ok = true;
                return t;
            }
        }
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
// Eight codes.
__device__ __forceinline__ u32x4 cvt8(uint32_t codes, float scale) {
    return {cvt2<0>(codes, scale), cvt2<1>(codes, scale), cvt2<2>(codes, scale), cvt2<3>(codes, scale)};
}
// Pair `sel` (a constant) of eight codes.
__device__ __forceinline__ uint32_t cvt_pair(uint32_t codes, float scale, int sel) {
    return sel == 0   ? cvt2<0>(codes, scale)
           : sel == 1 ? cvt2<1>(codes, scale)
           : sel == 2 ? cvt2<2>(codes, scale)
                      : cvt2<3>(codes, scale);
}
// The scale in byte i of four.
__device__ __forceinline__ float byte_scale(uint32_t bytes, int i) {
    return __uint_as_float((bytes >> 8 * i & 0xffu) << 23);
}

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
}

// The top 16 bits (a bf16) of two floats.
__device__ __forceinline__ uint32_t pack_top(float x, float y) {
    return perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
}
// What the bf16 that `mask` keeps of x leaves over.
__device__ __forceinline__ float rest(float x, uint32_t mask = 0xffff0000u) {
    return x - __uint_as_float(__float_as_uint(x) & mask);
}

// Row r's query.
__device__ __forceinline__ const float* att_query(const AttArgs& a, const AttItem& t, uint32_t head, uint32_t r) {
    return a.q + (uint64_t)(t.q0 + r / a.group) * a.q_stride + (uint64_t)(head * a.group + r % a.group) * a.dim;
}

// Eight values of a query row from dimension d on, scaled, as its three terms of
// eight bf16: the top 16 bits, then those of what they leave.
__device__ __forceinline__ void query_terms(const AttArgs& a, const float* q, uint32_t d, bool live,
                                            u32x4 (&term)[kAttTerms]) {
    float x[8];
    if (live && d + 8 <= a.dim) {
        const f32x4 u = (f32x4)*reinterpret_cast<const f32x4_a4*>(q + d);
        const f32x4 v = (f32x4)*reinterpret_cast<const f32x4_a4*>(q + d + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = u[i];
            x[4 + i] = v[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = live && d + i < a.dim ? q[d + i] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float u = x[2 * i] * a.scale_log2, v = x[2 * i + 1] * a.scale_log2;
#pragma unroll
        for (int k = 0; k < kAttTerms; ++k) {
            term[k][i] = pack_top(u, v);
            u = rest(u);
            v = rest(v);
        }
    }
}

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

// Where a step's tiles of 16 tokens lie: the page table through scalar loads,
// which have a counter of their own.  A tile past the end, or of a page that does
// not exist, is one of page 0 with no tokens: loads have no conditions on their
// way, so that a step's can be waited for while the next one's are in flight.
struct AttPages {
    typedef const __attribute__((address_space(4))) uint32_t* ScalarPtr;
    ScalarPtr table;
    const uint8_t* cache;
    uint32_t last, shift, kv_len, num_pages, page;
    uint64_t page_bytes;

    __device__ AttPages(const AttArgs& a, const AttItem& t, uint32_t head)
        : table((ScalarPtr)(uintptr_t)(a.table + (uint64_t)t.seq * a.max_pages)),
          cache(a.cache + (uint64_t)head * a.c.head_bytes),
          last(t.kv_len ? (t.kv_len - 1) >> a.c.shift : 0),
          shift(a.c.shift),
          kv_len(t.kv_len),
          num_pages(a.c.num_pages),
          page(a.c.page),
          page_bytes(a.c.page_bytes) {}

    __device__ uint32_t id(uint32_t tt) const { return table[min(tt * 16 >> shift, last)]; }
    // Tile tt of page `id`: its piece of the page, its tokens, the first's place.
    __device__ const uint8_t* at(uint32_t tt, uint32_t id, uint32_t* valid, uint32_t* t0) const {
        *valid = min(kv_len - min(kv_len, tt * 16), 16u);
        if (id >= num_pages) id = 0, *valid = 0;
        *t0 = (tt * 16) & (page - 1);
        return cache + (uint64_t)id * page_bytes;
    }
};

// V's four scale bytes of tokens first .. first + 3 of a tile that rows may not see
// all of: 1 for tokens that do not exist, and for NaN, which is reported.
__device__ __forceinline__ uint32_t finite_scales(uint32_t bytes, uint32_t first, uint32_t valid, bool* nan) {
    uint32_t out = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t b = bytes >> 8 * i & 0xffu;
        if (first + i >= valid) b = 127;
        if (b == kQ4NanScale) *nan = true, b = 127;
        out |= b << 8 * i;
    }
    return out;
}

// Blocks of V (bits) in which a token of tile tt that the lane's row sees is NaN.
// For steps that some rows see a part of: what their product takes instead is 1.
__device__ __forceinline__ uint32_t nan_blocks(const AttArgs& a, const AttPages& pages, uint32_t tt, uint32_t id,
                                            uint32_t limit) {
    uint32_t valid, t0, bits = 0;
    const uint8_t* base = pages.at(tt, id, &valid, &t0);
    for (uint32_t b = 0; b < a.c.nb; ++b)
        for (uint32_t i = 0; i < valid; ++i)
            if (base[q4_v_scale(a.c, t0 + i, b)] == kQ4NanScale && tt * 16 + i < limit) bits |= 1u << b;
    return bits;
}

// A row's running maximum, as what its probabilities are relative to.  It rises
// only when a score passes it by more than 2^8, so that sums and outputs are seldom
// rescaled; probabilities of up to 2^8 change no rounding.  (Scores that begin with
// minus the maximum would save a subtraction each: 2 % of a 64-row item, and 5 % lost
// where the registers spill.)
struct AttMax {
    static constexpr float kSlack = 8.0f;
    float base = 0.0f, limit = -__builtin_inff();  // limit: -inf before the first score, then base + kSlack

    __device__ float value() const { return limit == -__builtin_inff() ? limit : base; }
    // Scores of at most mx: what sums and outputs so far have to be multiplied by.
    __device__ float rise(float mx) {
        if (!(mx > limit)) return 1.0f;
        // before the first score there is nothing (or NaN) to rescale
        const float f = limit == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(base - mx);
        base = mx;
        limit = mx + kSlack;
        return f;
    }
};

// `kCount` values from dimension d on of the sequence's row rr, not yet divided by
// its sum l: to the output, or with its maximum m to the share's part.
template <uint32_t kRows, int kCount>
__device__ __forceinline__ void att_store(const AttArgs& a, const AttItem& t, uint32_t item, uint32_t head, uint32_t rr,
                                          float m, float l, uint32_t d, const float (&v)[kCount]) {
    if (t.splits > 1) {
        const uint32_t dp = 32 * a.c.nb;
        const uint64_t at = ((uint64_t)item * a.c.kv_heads + head) * kRows + (rr - t.first);
        if (d == 0) *reinterpret_cast<float2*>(a.part + at * 2) = make_float2(m, l);
        float* p = a.part + (uint64_t)a.items * a.c.kv_heads * kRows * 2 + at * dp + d;
#pragma unroll
        for (int i = 0; i < kCount; i += 4)
            if (d + i < dp) *reinterpret_cast<f32x4*>(p + i) = {v[i], v[i + 1], v[i + 2], v[i + 3]};
        return;
    }
    const float f = l == 0.0f ? 0.0f : 1.0f / l;
    float* p = a.out + ((uint64_t)(t.q0 + rr / a.group) * a.q_heads + head * a.group + rr % a.group) * a.dim + d;
#pragma unroll
    for (int i = 0; i < kCount; i += 4) {
        float u[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) u[k] = l == 0.0f ? 0.0f : v[i + k] * f;
        if (d + i + 4 <= a.dim) {
            *reinterpret_cast<f32x4_a4*>(p + i) = {u[0], u[1], u[2], u[3]};
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (d + i + k < a.dim) p[i + k] = u[k];
        }
    }
}

// What a lane (n = lane % 16, g = lane / 16) loads of one 16-token tile.
template <int NB>
struct AttKV {
    static constexpr int kC = NB < 4 ? 1 : NB / 4;  // 16-byte pieces
    uint32_t k[NB];   // token n's codes of group g, eight dimensions a dword
    u32x4 v[kC];      // four tokens of chunk n (or n / 2, or 2n and 2n + 1)
    uint32_t ks[kC];  // K's scale bytes
    uint32_t vs;      // V's scale bytes of tokens 4g .. 4g + 3
    uint32_t valid;   // tokens of the tile that exist
};

// NB: blocks of 32 dimensions that the tiles hold (2, 4 or 8), nb <= NB of them
// in use.  kSlot: rows of a matrix tile's 16 columns.  16: a product for each of
// three terms of q, and of p.  With 8 or 4 rows (a decode step's query heads) the
// terms lie side by side in the columns instead, column = slot * kSlot + row: one
// product takes two or all three, and the slots' scores are added across lanes.
// R: 16-row tiles of a wave.  An item's rows are kSlot, or with R = 2 four waves'
// 128: the waves deal out the rows, and where there are too few rows for four
// waves, the tokens, whose parts they join at the end.
template <int NB, int R, int kSlot>
struct AttShape {
    static constexpr uint32_t kWaveRows = kSlot < 16 ? kSlot : 16 * R;
    static constexpr uint32_t kRows = kSlot < 16 ? kSlot : 16 * R * kAttWaves;
    static constexpr int kSide = 16 / kSlot;                       // terms side by side
    static constexpr int kQ = (kAttTerms + kSide - 1) / kSide;     // products for a score
    static constexpr int kP = kQ;                                  // products for an output
};

// A step, v_mfma_f32_16x16x32_bf16: for S^T a lane holds token n's dimensions of
// group g (K's codes as they lie, 16 bytes at head_dim 128; which eight of them
// meet in one product is free, q's operand is taken alike) and gets tokens 4g ..
// 4g + 3 of row n, for two tiles; for O^T those are its eight tokens.
//
// kRaise: a wave's products go before other waves' softmax (s_setprio).  45 x 8192, 4
// query heads on each of 8 key heads: 52.3 -> 50.9 us, 8 on each of 64 sequences 78 ->
// 73; 64-row items after long contexts 5 .. 8 % (512 after 4096: 157 -> 148), but not 16
// rows a sequence (65 -> 71) nor prompts of their own keys (1024: 37 -> 40), nor 256
// dimensions (152 -> 171).  A branch on it would cost as much as it gives.
template <int NB, int R, int kSlot, int kPerSimd, bool kRaise>
__global__ __launch_bounds__(kAttBlock) __attribute__((amdgpu_waves_per_eu(kPerSimd, kPerSimd)))
void att_kernel(AttArgs a) {
    using Shape = AttShape<NB, R, kSlot>;
    constexpr uint32_t kRows = Shape::kRows, kWaveRows = Shape::kWaveRows;
    constexpr int kQ = Shape::kQ, kP = Shape::kP, kC = AttKV<NB>::kC, kSide = Shape::kSide;
    constexpr int kJ = 2 * NB;  // dimensions of a lane's part of a row, and O tiles
    const uint32_t lane = threadIdx.x % kWave, n = lane % 16, g = lane / 16;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave));
    // Key heads change fastest: workgroups go round the 8 XCDs, and every XCD gets
    // its part of the items, of which the last may be empty.
    const uint32_t head = blockIdx.x % a.c.kv_heads, item = a.item0 + blockIdx.x / a.c.kv_heads;
    const AttItem t = att_item<kRows, false>(a, item);
    if (!t.ok) return;
    const uint32_t nb = a.c.nb;
    // The item's share of its steps: [lo, hi).
    const uint32_t steps = att_steps(att_limit(a, t, min(t.first + kRows, t.rows) - 1));
    const uint32_t lo = t.splits > 1 ? t.split * t.chunk : 0, hi = t.splits > 1 ? min(lo + t.chunk, steps) : steps;
    if (t.splits > 1 && lo >= hi) return;  // the joining kernel knows
    // The waves' rows: one, two or four groups of them; the waves of a group share
    // its tokens.
    const uint32_t left = min(t.rows - t.first, kRows);
    const uint32_t groups = left <= kWaveRows ? 1 : left <= 2 * kWaveRows ? 2 : 4;
    const uint32_t stride = kAttWaves / groups;
    const uint32_t r0 = t.first + (wave % groups) * kWaveRows;  // the wave's first row
    const uint32_t r1 = min(r0 + kWaveRows, t.rows);            // its end; r0 or less: no rows
    const uint32_t min_limit = att_limit(a, t, min(r0, t.rows - 1));
    const uint32_t end = r0 < r1 ? min(hi, att_steps(att_limit(a, t, r1 - 1))) : 0;

    // q's third term lies in LDS where the registers would not hold it (4 x 4096
    // tokens, 32 + 8 heads of 128: 1295 -> 1193 us, the spills gone).
    constexpr bool kPark = kSlot == 16 && R == 2 && NB == 4;
    constexpr int kHeldQ = kPark ? kQ - 1 : kQ;
    union Shared {
        float so[kAttWaves][16][16 * kJ + 4];
        u32x4 q[kPark ? kAttWaves : 1][R][NB][kWave];
        __device__ Shared() {}
    };
    __shared__ __attribute__((aligned(16))) Shared shared;
    const uint32_t slot = n / kSlot;
    // What a lane of slot 1, and of slot 2, leaves out of a probability before its own term.
    const uint32_t cut1 = kSlot < 16 && slot >= 1 ? 0xffff0000u : 0, cut2 = kSlot < 16 && slot >= 2 ? 0xffff0000u : 0;
    const uint32_t slot1 = slot ? 0xffffffffu : 0;
    uint32_t limit[R];
    u32x4 qf[R][kHeldQ][NB];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const uint32_t row = r0 + 16 * r + n % kSlot;
        const bool live = row < r1;
        limit[r] = live ? att_limit(a, t, row) : 0;
        const float* qp = att_query(a, t, head, live ? row : 0);
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            u32x4 term[kAttTerms];
            query_terms(a, qp, g * 8 * NB + 8 * j, live, term);
#pragma unroll
            for (int k = 0; k < kQ; ++k) {
                u32x4 w = {0, 0, 0, 0};
#pragma unroll
                for (int at = 0; at < kSide; ++at)
                    if (k * kSide + at < kAttTerms && slot == (uint32_t)at) w = term[k * kSide + at];
                if (k < kHeldQ) qf[r][k][j] = w;
                else shared.q[wave][r][j][lane] = w;
            }
        }
    }

    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    const float ninf = -__builtin_inff();
    f32x4 o[R][kJ];
    AttMax top[R];
    float l[R];
    uint32_t poison[R];  // blocks of V in which the row sees NaN that others do not
#pragma unroll
    for (int r = 0; r < R; ++r) {
        l[r] = 0.0f;
        poison[r] = 0;
#pragma unroll
        for (int j = 0; j < kJ; ++j) o[r][j] = zero;
    }

    // Blocks past nb are read from the last one: q is zero there, and what they add
    // to the output is not stored.
    const AttPages pages(a, t, head);
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
        uint32_t t0;
        const uint8_t* base = pages.at(tt, page, &x.valid, &t0);
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

    auto work = [&](uint32_t step, AttKV<NB> (&cur)[2], const uint32_t (&page)[2]) {
        if constexpr (kRaise) __builtin_amdgcn_s_setprio(1);
        // Scores, in powers of two: tokens 4g + i of both tiles.
        f32x4 s[R][2];
#pragma unroll
        for (int r = 0; r < R; ++r) s[r][0] = s[r][1] = zero;
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            u32x4 q3[R];
            if constexpr (kPark)
#pragma unroll
                for (int r = 0; r < R; ++r) q3[r] = shared.q[wave][r][j][lane];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const u32x4 kf = cvt8(cur[x].k[j], byte_scale(cur[x].ks[j / 4], 0));
#pragma unroll
                for (int k = kQ - 1; k >= 0; --k)
#pragma unroll
                    for (int r = 0; r < R; ++r) s[r][x] = mfma(kf, k < kHeldQ ? qf[r][k < kHeldQ ? k : 0][j] : q3[r], s[r][x]);
            }
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
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const uint32_t have = min(limit[r], at + 16 * x + cur[x].valid);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (at + 16 * x + 4 * g + i >= have) s[r][x][i] = ninf;
                }
                cur[x].vs = finite_scales(cur[x].vs, 4 * g, cur[x].valid, &nan_v);
            }
        }
        if constexpr (kRaise) __builtin_amdgcn_s_setprio(0);
        // Running maximum, probabilities and their sum; bf16 terms.
        u32x4 pf[R][kP];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float mx = fmaxf(fmaxf(fmaxf(s[r][0][0], s[r][0][1]), fmaxf(s[r][0][2], s[r][0][3])),
                             fmaxf(fmaxf(s[r][1][0], s[r][1][1]), fmaxf(s[r][1][2], s[r][1][3])));
            if (__any(mx > top[r].limit)) {
                mx = fmaxf(mx, __shfl_xor(mx, 16, kWave));
                mx = fmaxf(mx, __shfl_xor(mx, 32, kWave));
                const float f = top[r].rise(mx);
                l[r] *= f;
#pragma unroll
                for (int j = 0; j < kJ; ++j) o[r][j] *= f;
            }
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    const float p0 = __builtin_amdgcn_exp2f(s[r][x][i] - top[r].base);
                    const float p1 = __builtin_amdgcn_exp2f(s[r][x][i + 1] - top[r].base);
                    l[r] += p0 + p1;
                    // the lane's term (slot 3's column is not read)
                    float u0 = rest(p0, cut1), u1 = rest(p1, cut1);
                    if constexpr (kSlot == 4) u0 = rest(u0, cut2), u1 = rest(u1, cut2);
#pragma unroll
                    for (int k = 0; k < kP; ++k) {
                        pf[r][k][2 * x + i / 2] = pack_top(u0, u1);
                        u0 = rest(u0);
                        u1 = rest(u1);
                    }
                    if constexpr (kSlot == 8) pf[r][1][2 * x + i / 2] &= slot1;  // the third term is slot 1's
                }
        }
        if constexpr (kRaise) __builtin_amdgcn_s_setprio(1);
        // V: four dwords a tile are four tokens x eight dimensions; an operand is
        // eight tokens of one dimension.
        float vsc[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) vsc[i] = byte_scale(cur[i >> 2].vs, i & 3);
#pragma unroll
        for (int p = 0; p < NB; ++p) {  // pair of dimensions 2p, 2p + 1
            uint32_t v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                uint32_t code = cur[i >> 2].v[NB == 8 ? p >> 2 : 0][i & 3];
                if (NB == 2) code >>= (n & 1) * 16;  // the lane's four dimensions of the chunk
                v[i] = cvt_pair(code, vsc[i], p & 3);
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
        if constexpr (kRaise) __builtin_amdgcn_s_setprio(0);
        if (!whole && __any(nan_v)) {
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int r = 0; r < R; ++r) poison[r] |= nan_blocks(a, pages, 2 * step + x, page[x], limit[r]);
        }
    };

    // Two steps in turn: one's loads are in flight while the other is worked on,
    // the pages of the one after that on their way.
    uint32_t step = lo + wave / groups;
    if (step < end) {
        AttKV<NB> kv[2][2];
        uint32_t page[2][2], ahead[2];
        auto fetch = [&](uint32_t st, int to) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                page[to][x] = ahead[x];
                load(2 * st + x, ahead[x], kv[to][x]);
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) ahead[x] = pages.id(2 * (st + stride) + x);
        };
        ahead[0] = pages.id(2 * step);
        ahead[1] = pages.id(2 * step + 1);
        fetch(step, 0);
        for (;;) {
            fetch(step + stride, 1);
            work(step, kv[0], page[0]);
            step += stride;
            if (step >= end) break;
            fetch(step + stride, 0);
            work(step, kv[1], page[1]);
            step += stride;
            if (step >= end) break;
        }
    }

    // Lane (n, g) has dimensions kJ (4g + i) + j of row n in o[.][j][i].
#pragma unroll
    for (int r = 0; r < R; ++r) {
        l[r] += __shfl_xor(l[r], 16, kWave);
        l[r] += __shfl_xor(l[r], 32, kWave);
        if (poison[r]) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (poison[r] >> NB * (4 * g + i) / 16 & 1)
#pragma unroll
                    for (int j = 0; j < kJ; ++j) o[r][j][i] = __uint_as_float(0x7fc00000u);
        }
    }
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
                    att_store<kRows>(a, t, item, head, row, top[r].value(), l[r], kJ * (4 * g + i), v);
                }
            }
        }
        return;
    }
    // Join the waves of a group: to the common maximum, then add (and the terms'
    // columns to the first's).
    __shared__ float sm[kAttWaves][16], sl[kAttWaves][16];
    auto& so = shared.so;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        __syncthreads();
        if (g == 0) {
            sm[wave][n] = top[r].value();
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
            float mm = ninf, ll = 0.0f, v[4] = {0.f, 0.f, 0.f, 0.f};
            for (uint32_t w = gr; w < kAttWaves; w += groups) mm = fmaxf(mm, sm[w][row]);
            for (uint32_t w = gr; w < kAttWaves; w += groups) {
                // a wave that saw nothing holds zeros (or NaN, which stays)
                const float f = sm[w][row] == ninf ? 1.0f : __builtin_amdgcn_exp2f(sm[w][row] - mm);
                ll += sl[w][row] * f;
                f32x4 u = *reinterpret_cast<const f32x4*>(&so[w][row][d]);
#pragma unroll
                for (int at = 1; at < kSide && at < kAttTerms; ++at)
                    u += *reinterpret_cast<const f32x4*>(&so[w][row + at * kSlot][d]);
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] += u[k] * f;
            }
            att_store<kRows>(a, t, item, head, rr, mm, ll, d, v);
        }
    }
}

// Four dimensions of row rr, their sum l.
__device__ __forceinline__ void join_store(const AttArgs& a, const AttItem& t, uint32_t head, uint32_t rr, uint32_t d,
                                           float l, f32x4 v) {
    float* out = a.out + ((uint64_t)(t.q0 + rr / a.group) * a.q_heads + head * a.group + rr % a.group) * a.dim + d;
    const float f = 1.0f / l;
    f32x4 u;
#pragma unroll
    for (int k = 0; k < 4; ++k) u[k] = l == 0.0f ? 0.0f : v[k] * f;
    if (d + 4 <= a.dim) {
        *reinterpret_cast<f32x4_a4*>(out) = (f32x4_a4)u;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (d + k < a.dim) out[k] = u[k];
    }
}

// What a share's sum and outputs are multiplied by, its maximum m, all shares' mm:
// one that saw nothing holds zeros (or NaN, which stays).
__device__ __forceinline__ float join_factor(float m, float mm) {
    return m == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(m - mm);
}

// The shares of `count` rows of a tile from row `from` on.
struct JoinRows {
    AttItem t;
    uint32_t head, from, count, used, dp;
    uint64_t next;     // rows to the next share's
    const float2* ml;  // maximum and sum of the first row in the first share
    const float* out;  // its outputs
};

template <uint32_t kRows, uint32_t kParts>
__device__ __forceinline__ JoinRows join_rows(const AttArgs& a) {
    JoinRows j;
    const uint32_t tile = blockIdx.x / kParts;
    j.from = blockIdx.x % kParts * (kRows / kParts);
    j.head = tile % a.c.kv_heads;
    j.t = att_item<kRows, true>(a, tile / a.c.kv_heads);
    const AttItem& t = j.t;
    j.count = !t.ok || t.splits == 1 || t.first + j.from >= t.rows ? 0 : min(kRows / kParts, t.rows - t.first - j.from);
    if (j.count == 0) return j;
    const uint32_t last_row = min(t.first + kRows, t.rows) - 1;
    j.used = (att_steps(att_limit(a, t, last_row)) + t.chunk - 1) / t.chunk;
    j.dp = 32 * a.c.nb;
    j.next = (uint64_t)a.c.kv_heads * kRows;
    const uint64_t row0 = ((uint64_t)t.item * a.c.kv_heads + j.head) * kRows + j.from;
    j.ml = reinterpret_cast<const float2*>(a.part) + row0;
    j.out = a.part + (uint64_t)a.items * a.c.kv_heads * kRows * 2 + row0 * j.dp;
    return j;
}

// Joins the shares of a tile: a thread has four dimensions of a row and goes over
// the shares, kAhead of them in flight.
template <uint32_t kRows>
struct AttJoin {
    static constexpr uint32_t kThreads = kRows <= 8 ? 128 : 256;
    static constexpr uint32_t kParts = kRows <= 8 ? 1 : kRows / 16;  // workgroups of a tile
    static constexpr int kAhead = 8;
};

template <uint32_t kRows>
__global__ __launch_bounds__(AttJoin<kRows>::kThreads) void att_join_kernel(AttArgs a) {
    constexpr int kAhead = AttJoin<kRows>::kAhead;
    const JoinRows j = join_rows<kRows, AttJoin<kRows>::kParts>(a);
    const uint32_t quads = j.dp / 4, at_once = AttJoin<kRows>::kThreads / quads;
    if (j.count == 0 || threadIdx.x >= at_once * quads) return;
    const uint32_t d = threadIdx.x % quads * 4;
    for (uint32_t row = threadIdx.x / quads; row < j.count; row += at_once) {
        const float ninf = -__builtin_inff();
        float mm = ninf, ll = 0.0f;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        for (uint32_t z0 = 0; z0 < j.used; z0 += kAhead) {
            float2 u[kAhead];
            f32x4 w[kAhead];
#pragma unroll
            for (int z = 0; z < kAhead; ++z) {
                const uint64_t at = min(z0 + z, j.used - 1) * j.next + row;
                u[z] = j.ml[at];
                w[z] = *reinterpret_cast<const f32x4*>(j.out + at * j.dp + d);
            }
            float top = mm;
#pragma unroll
            for (int z = 0; z < kAhead; ++z) top = fmaxf(top, u[z].x);
            const float f0 = join_factor(mm, top);
            mm = top;
            ll *= f0;
            v *= f0;
#pragma unroll
            for (int z = 0; z < kAhead; ++z)
                if (z0 + z < j.used) {
                    const float f = join_factor(u[z].x, mm);
                    ll += u[z].y * f;
                    v += w[z] * f;
                }
        }
        join_store(a, j.t, j.head, j.t.first + j.from + row, d, ll, v);
    }
}

// The same for many shares of few tiles: a workgroup has one row, its threads the
// shares' maxima and sums, then four dimensions and every kth share each.
template <uint32_t kRows>
__global__ __launch_bounds__(kAttBlock) void att_join_wide_kernel(AttArgs a) {
    constexpr uint32_t kEach = kAttMaxSplits / kAttBlock;
    __shared__ float factor[kAttMaxSplits], one[kAttWaves];
    __shared__ f32x4 red[kAttBlock];
    const JoinRows j = join_rows<kRows, kRows>(a);
    if (j.count == 0) return;
    const uint32_t wave = threadIdx.x / kWave;
    const float ninf = -__builtin_inff();
    float2 u[kEach];
    float mm = ninf, ll = 0.0f;
#pragma unroll
    for (uint32_t k = 0; k < kEach; ++k) {
        const uint32_t z = threadIdx.x + k * kAttBlock;
        u[k] = z < j.used ? j.ml[z * j.next] : make_float2(ninf, 0.0f);
        mm = fmaxf(mm, u[k].x);
    }
#pragma unroll
    for (int x = 1; x < kWave; x *= 2) mm = fmaxf(mm, __shfl_xor(mm, x, kWave));
    one[wave] = mm;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kAttWaves; ++w) mm = fmaxf(mm, one[w]);
    __syncthreads();
#pragma unroll
    for (uint32_t k = 0; k < kEach; ++k) {
        const float f = join_factor(u[k].x, mm);
        factor[threadIdx.x + k * kAttBlock] = f;
        ll += u[k].y * f;
    }
#pragma unroll
    for (int x = 1; x < kWave; x *= 2) ll += __shfl_xor(ll, x, kWave);
    one[wave] = ll;
    __syncthreads();
    ll = one[0];
#pragma unroll
    for (int w = 1; w < kAttWaves; ++w) ll += one[w];
    const uint32_t quads = j.dp / 4, groups = kAttBlock / quads, gr = threadIdx.x / quads, d = threadIdx.x % quads * 4;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (gr < groups) {
#pragma unroll 8
        for (uint32_t z = gr; z < j.used; z += groups)
            v += *reinterpret_cast<const f32x4*>(j.out + z * j.next * j.dp + d) * factor[z];
    }
    red[threadIdx.x] = v;
    __syncthreads();
    if (gr != 0) return;
    for (uint32_t k = 1; k < groups; ++k) v += red[threadIdx.x + k * quads];
    join_store(a, j.t, j.head, j.t.first + j.from, d, ll, v);
}

struct AttPlan {
    uint32_t rows;  // kRows: 4, 8 (kSlot), 64 or 128 (kSlot 16)
    uint32_t tiles, items, target;
    bool wide;       // many shares of a tile
    bool search;     // many sequences
    bool raise;      // 64-row items: most keys are older than the new tokens
    uint64_t bytes;  // workspace
};

// Sizes decide what the device cannot wait to see; lengths are not known here.
//
// Rows.  Prompts whose 128-row items fit on the chip all at once (two workgroups a
// CU) take 64-row items: they end evenly (2048 tokens, 32 + 8 heads of 128: 105 ->
// 85 us; 512 tokens 30 -> 18).  With more, 128 rows need a key's and a value's
// conversion half as often (4 x 4096 of 16 heads of 64: 152 us, with 64 rows 160).
//
// Cut.  Keys are cut where the tiles are fewer than the workgroups that the chip
// holds at once.  45 decode steps over up to 8192 tokens, 8 key heads: 67 -> 53 us;
// 96 of them: 108 us, cut 114; 4 x 256 tokens after 32768: 1031 -> 608 us.  Below
// 2048 tokens the second kernel costs more than the shares save (1 x 1024: 10.4 us,
// cut 12.1; 1 x 2048: 12.0 us, uncut 15.8).  From 16384 tokens on up to twice as many
// tiles are cut, finer, for sequences of very different lengths (3 x 1024 tokens
// after 32768: 2211 -> 1487 us; 80 x 20000, 8 query heads a key head: 244 -> 206;
// equal lengths lose 5 % at most: 190 x 17000 603 -> 631).
//
// Share.  At least 8 steps, two for each wave, and 16 or 32 of long sequences (worked
// out from the lengths, att_item): 1 x 2048 11.3 us (16: 12.5), 1 x 16384 17.0 (16:
// 14.9), 1 x 65536 26.7 (32: 24.4; 48: 24.8).
//
// Search.  Every workgroup looks through the sequences up to its own, 256 at a time;
// past 2048 it searches, in a numbering with gaps (4000 x 512: 1479 -> 711 us, 1000 x
// 1024: 202 -> 233).
//
// Join.  With more than 8 shares a tile a workgroup joins one row (1 x 131072, 8
// query heads on 1: 145 -> 36 us); with fewer all rows of a tile do (45 x 8192: 48
// us, 53 with a workgroup a row).
static int att_plan(uint64_t num_seqs, uint64_t tokens, uint64_t q_heads, uint64_t kv_heads, uint64_t page_size,
                    uint64_t max_pages, uint32_t nb, AttPlan* p) {
    const uint64_t group = q_heads / kv_heads, rows = tokens * group;
    p->rows = rows <= 4 * num_seqs                                                       ? 4
              : rows <= 8 * num_seqs                                                     ? 8
              : rows <= 16 * num_seqs || nb > 4 || rows / 128 * kv_heads <= 2 * kAttCus ? 64
                                                                                         : 128;
    const uint64_t some = std::min(num_seqs, tokens);  // sequences with new tokens, at most
    const uint64_t want = (p->rows == 4 && nb <= 4 ? 3 : 2) * kAttCus;  // workgroups that the chip holds at once
    const uint64_t busy = std::max(some, rows / p->rows);
    const uint64_t shares = max_pages * page_size / (kAttMinChunk * kAttStep);  // of the longest sequence
    const uint64_t more = shares >= 64 ? 2 : 1;
    const bool cut = busy * kv_heads < more * want && shares >= 8 && num_seqs <= 4096;
    p->search = !cut && num_seqs > 2048;
    const uint64_t tiles = rows / p->rows + (p->search ? num_seqs : some);
    if (tiles > 0x3fffffull) return KORE_HIP_ERR_OVERFLOW;
    p->target = cut ? (uint32_t)std::min<uint64_t>({std::max((want + kv_heads - 1) / kv_heads, 2 * more * busy),
                                                    tiles * shares, kAttMaxSplits})
                    : 0;
    p->wide = p->target > 8 * tiles;
    p->raise = rows > 16 * num_seqs && nb <= 4 && 2 * tokens < num_seqs * max_pages * page_size;
    p->tiles = (uint32_t)tiles;
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

enum class AttPass { kItems, kJoin, kJoinWide };

// count: items or tiles.
template <int NB, int R, int kSlot, int kPerSimd, bool kRaise = kSlot < 16 && NB < 8>
static void att_launch_shape(const AttArgs& a, AttPass pass, uint32_t count, hipStream_t s) {
    constexpr uint32_t kRows = AttShape<NB, R, kSlot>::kRows;
    const uint32_t x = count * a.c.kv_heads;
    if (pass == AttPass::kItems)
        hipLaunchKernelGGL((att_kernel<NB, R, kSlot, kPerSimd, kRaise>), dim3(x), dim3(kAttBlock), 0, s, a);
    else if (pass == AttPass::kJoin)
        hipLaunchKernelGGL((att_join_kernel<kRows>), dim3(x * AttJoin<kRows>::kParts), dim3(AttJoin<kRows>::kThreads), 0,
                           s, a);
    else
        hipLaunchKernelGGL((att_join_wide_kernel<kRows>), dim3(x * kRows), dim3(kAttBlock), 0, s, a);
}

// kPerSimd: the waves that a SIMD's registers hold.  With one fewer 64-row items of 64
// dimensions took 107 us where they take 96, 8-row ones 62 where 57 (45 x 8192, 40 + 8
// heads of 96); one more spills.
static void att_launch(const AttArgs& a, const AttPlan& p, AttPass pass, uint32_t count, hipStream_t s) {
    auto launch = [&](auto blocks) {
        constexpr int NB = decltype(blocks)::value;
        constexpr int kMid = NB == 8 ? 1 : NB == 4 ? 2 : 3;
        if (p.rows == 4) att_launch_shape<NB, 1, 4, NB == 8 ? 2 : 3>(a, pass, count, s);
        else if (p.rows == 8) att_launch_shape<NB, 1, 8, NB == 8 ? 1 : NB == 4 ? 3 : 4>(a, pass, count, s);
        else if (p.rows == 64 && p.raise && pass == AttPass::kItems)
            att_launch_shape<NB, 1, 16, kMid, (NB < 8)>(a, pass, count, s);
        else if (p.rows == 64) att_launch_shape<NB, 1, 16, kMid>(a, pass, count, s);
        else if constexpr (NB < 8) att_launch_shape<NB, 2, 16, 2>(a, pass, count, s);
    };
    if (a.c.nb <= 2) launch(std::integral_constant<int, 2>());
    else if (a.c.nb <= 4) launch(std::integral_constant<int, 4>());
    else launch(std::integral_constant<int, 8>());
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
    if (p.bytes && (att_overlap(workspace, p.bytes, q, ((tokens - 1) * a.q_stride + row) * 4) ||
                    att_overlap(workspace, p.bytes, cache, bytes) ||
                    att_overlap(workspace, p.bytes, page_table, num_seqs * max_pages * 4) ||
                    att_overlap(workspace, p.bytes, kv_lens, num_seqs * 4) ||
                    att_overlap(workspace, p.bytes, q_starts, num_seqs * 4 + 4)))
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
    a.search = p.search;
    a.scale_log2 = (float)((double)scale * 1.4426950408889634);
    a.causal = causal != 0;
    // A launch holds fewer than 2^32 threads: items in bands.
    const uint32_t band = (uint32_t)std::max<uint64_t>(1, 0x400000u / kv_heads);
    for (a.item0 = 0; a.item0 < p.items; a.item0 += band) {
        att_launch(a, p, AttPass::kItems, std::min(band, p.items - a.item0), (hipStream_t)stream);
        const int rc = launch_status();
        if (rc != KORE_HIP_OK) return rc;
    }
    if (p.target) {  // few tiles, or their keys would not be cut
        att_launch(a, p, p.wide ? AttPass::kJoinWide : AttPass::kJoin, p.tiles, (hipStream_t)stream);
        return launch_status();
    }
    return KORE_HIP_OK;
}
