// attention_q4.hip -- softmax(scale q k^T) v over the paged 4-bit cache, for
// ragged sequences with any number of new tokens each.
//
// One pass over the keys with the running maximum and sum of the softmax; no
// scores in memory.  The rows of one key head are its query heads times the
// sequence's new tokens: row r = token * group + head, 16 to a matrix tile.
//
// Arithmetic.  A cached value is a code times a power of two, exact in bf16, so
// the matrix cores' bf16 form loses nothing on the cache's side.  A query value
// (times scale * log2 e, one f32 rounding) is cut into three bf16 terms of 8
// bits each, which is all of its 24: every product q * k is exact and sums are
// f32.  A probability is two bf16 terms rounded to nearest: it is off by at
// most 2^-18 of itself, half of what a term of 16 bits leaves, next to the few
// f32 roundings in the score that it is the exponential of; the row's sum takes
// the f32 value.
//
// Layout of a step (32 tokens, v_mfma_f32_16x16x32_bf16; n = lane % 16,
// g = lane / 16):
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

#include "q4.hpp"

namespace kore {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kAttBlock = 256;
constexpr int kAttWaves = kAttBlock / kWave;
constexpr uint32_t kAttStep = 32;      // tokens of a step
constexpr uint32_t kAttCombine = 256;  // threads of the joining kernel

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
    uint32_t num_seqs, q_heads, group, max_pages, dim, tiles, tile0, splits;
    float scale_log2;
    int causal;
    Q4Cache c;
};

// A tile: `rows` consecutive rows of one sequence and key head.
struct AttTile {
    uint32_t seq, q0, q_len, kv_len, first;  // first: its first row in the sequence
    uint32_t rows;                           // rows of the sequence
    bool ok;
};

// Sequence s owns tiles from start_s * group / kRows + s on: its
// ceil(len * group / kRows) tiles end before the next sequence's first, so a
// tile's number alone names it.  Tiles between are empty.
template <uint32_t kRows>
__device__ __forceinline__ AttTile att_tile(const AttArgs& a, uint32_t tile) {
    AttTile t = {};
    uint32_t before = 0;
    for (uint32_t s0 = 0; s0 < a.num_seqs; s0 += kWave) {
        const uint32_t s = s0 + lane_id();
        bool le = false;
        if (s < a.num_seqs) {
            const uint64_t st = a.starts[s] < a.tokens ? a.starts[s] : a.tokens;
            le = st * a.group / kRows + s <= tile;
        }
        const uint64_t m = __ballot(le);
        before += (uint32_t)__popcll(m);
        if (m != ~0ull) break;
    }
    if (before == 0) return t;
    before = (uint32_t)__builtin_amdgcn_readfirstlane((int)before);
    t.seq = before - 1;
    const uint32_t lim = (uint32_t)a.tokens;
    t.q0 = min(a.starts[t.seq], lim);
    const uint32_t q1 = min(a.starts[t.seq + 1], lim);
    if (q1 <= t.q0) return t;
    t.q_len = q1 - t.q0;
    const uint64_t rows = (uint64_t)t.q_len * a.group;
    const uint64_t base = (uint64_t)t.q0 * a.group / kRows + t.seq;
    const uint64_t first = (tile - base) * kRows;
    if (first >= rows) return t;
    const uint64_t cap = (uint64_t)a.max_pages << a.c.shift;
    const uint32_t len = a.lens[t.seq];
    t.kv_len = len < cap ? len : (uint32_t)cap;
    if (a.c.num_pages == 0) t.kv_len = 0;
    t.first = (uint32_t)first;
    t.rows = (uint32_t)rows;
    t.ok = true;
    return t;
}

// Keys that row r of the sequence sees: all, or those up to its own position,
// the last new token sitting at kv_len - 1.
__device__ __forceinline__ uint32_t att_limit(const AttArgs& a, const AttTile& t, uint32_t r) {
    if (!a.causal) return t.kv_len;
    const uint32_t after = t.q_len - 1 - r / a.group;
    return t.kv_len > after ? t.kv_len - after : 0;
}

// Steps of a tile that sees `limit` keys, and their share for one split.
__device__ __forceinline__ uint32_t att_steps(uint32_t limit) { return (limit + kAttStep - 1) / kAttStep; }
__device__ __forceinline__ uint32_t att_share(uint32_t steps, uint32_t splits) { return (steps + splits - 1) / splits; }

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

// What a lane loads of one 16-token tile.
template <int NB>
struct AttKV {
    static constexpr int kV = NB < 4 ? 4 : NB;
    uint32_t k[NB];  // token n's codes of group g, eight dimensions a dword
    uint32_t v[kV];  // four tokens of chunk n (or half of n / 2, or 2n and 2n + 1)
    uint32_t ks;     // K's scale bytes: one block's, or two blocks'
    uint32_t vs;     // V's scale bytes of tokens 4g .. 4g + 3
    uint32_t valid;  // tokens of the tile that exist
};

// NB: blocks of 32 dimensions that the tiles hold (2, 4 or 8), nb <= NB of them
// in use; R: 16-row tiles of a wave; Split: the workgroup's waves share the
// rows and deal out the tokens, else each wave has rows of its own.
template <int NB, int R, bool Split>
__global__ __launch_bounds__(kAttBlock) void att_kernel(AttArgs a) {
    constexpr uint32_t kRows = 16u * R * (Split ? 1 : kAttWaves);
    constexpr int kJ = 2 * NB;                 // dimensions of a lane's O rows, O tiles
    constexpr int kV = AttKV<NB>::kV;
    const uint32_t lane = threadIdx.x % kWave, n = lane % 16, g = lane / 16;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave));
    const uint32_t tile_id = a.tiles - 1 - a.tile0 - blockIdx.x;  // rows that see the most keys first
    const uint32_t head = blockIdx.y, split = blockIdx.z;
    const AttTile t = att_tile<kRows>(a, tile_id);
    if (!t.ok) return;
    const uint32_t nb = a.c.nb;
    const uint32_t r0 = t.first + (Split ? 0 : wave * 16 * R);  // the wave's first row
    const uint32_t last_row = min(t.first + kRows, t.rows) - 1;
    const bool have = r0 < t.rows;

    // Tokens of this split, then of this wave.
    const uint32_t steps = att_steps(att_limit(a, t, last_row)), share = att_share(steps, a.splits);
    const uint32_t lo = split * share, hi = min(lo + share, steps);
    if (a.splits > 1 && lo >= hi) return;  // the joining kernel knows
    uint32_t end = hi;
    const uint32_t min_limit = att_limit(a, t, min(r0, t.rows - 1));
    if (!Split) end = have ? min(hi, att_steps(att_limit(a, t, min(r0 + 16 * R, t.rows) - 1))) : 0;

    uint32_t limit[R];
    u32x4 qf[R][3][NB];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const uint32_t row = r0 + 16 * r + n;
        const bool live = row < t.rows;
        limit[r] = live ? att_limit(a, t, row) : 0;
        const uint32_t tok = live ? t.q0 + row / a.group : 0, hd = head * a.group + row % a.group;
        const float* qp = a.q + (uint64_t)tok * a.q_stride + (uint64_t)hd * a.dim;
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
#pragma unroll
                for (int term = 0; term < 3; ++term) {  // the top 16 bits, then what they leave
                    const uint32_t ub = __float_as_uint(u), vb = __float_as_uint(v);
                    qf[r][term][j][i] = perm(vb, ub, 0x07060302u);
                    u -= __uint_as_float(ub & 0xffff0000u);
                    v -= __uint_as_float(vb & 0xffff0000u);
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

    const uint32_t* table = a.table + (uint64_t)t.seq * a.max_pages;
    // Tile tt's place in the cache; a page that does not exist has no tokens.
    auto place = [&](uint32_t tt, uint32_t* valid) {
        const uint32_t at = tt * 16;
        uint32_t page = 0, v = 0;
        if (at < t.kv_len) {
            page = (uint32_t)__builtin_amdgcn_readfirstlane((int)table[at >> a.c.shift]);
            v = min(t.kv_len - at, 16u);
            if (page >= a.c.num_pages) page = 0, v = 0;
        }
        *valid = v;
        return a.cache + (uint64_t)page * a.c.page_bytes + (uint64_t)head * a.c.head_bytes;
    };
    auto load = [&](uint32_t tt, AttKV<NB>& x) {
        const uint8_t* base = place(tt, &x.valid);
        const uint32_t t0 = (tt * 16) & (a.c.page - 1), np = a.c.page * nb;
        const uint8_t* kp = base + (t0 + n) * nb * 16 + g * 4 * NB;
        const uint8_t* vp = base + np * 16 + t0 * nb * 16;
        const uint8_t* ksp = base + np * 32 + (t0 + n) * nb;
        const uint8_t* vsp = base + np * 33 + t0 * nb + 4 * g;
        x.ks = x.vs = 0x7f7f7f7fu;
#pragma unroll
        for (int j = 0; j < NB; ++j) x.k[j] = 0;
#pragma unroll
        for (int j = 0; j < kV; ++j) x.v[j] = 0;
        if constexpr (NB == 2) {
            if (g < 2 * nb) {
                const u32x2 u = *reinterpret_cast<const u32x2*>(kp);
                x.k[0] = u.x;
                x.k[1] = u.y;
                x.ks = ksp[g >> 1];
            }
            if (n >> 1 < 4 * nb) {
                const u32x4 u = *reinterpret_cast<const u32x4*>(vp + (g * 4 * nb + (n >> 1)) * 16);
#pragma unroll
                for (int i = 0; i < 4; ++i) x.v[i] = u[i] >> (n & 1) * 16;  // the lane's four dimensions
                x.vs = *reinterpret_cast<const uint32_t*>(vsp + (n >> 3) * 16);
            }
        } else {
#pragma unroll
            for (int c = 0; c < NB / 4; ++c) {
                const uint32_t block = g * (NB / 4) + c;
                if (block < nb) {
                    const u32x4 u = *reinterpret_cast<const u32x4*>(kp + 16 * c);
#pragma unroll
                    for (int i = 0; i < 4; ++i) x.k[4 * c + i] = u[i];
                    x.ks = c ? (x.ks & 0xffu) | (uint32_t)ksp[block] << 8 : ksp[block];
                }
                const uint32_t chunk = n * (NB / 4) + c;
                if (chunk < 4 * nb) {
                    const u32x4 u = *reinterpret_cast<const u32x4*>(vp + (g * 4 * nb + chunk) * 16);
#pragma unroll
                    for (int i = 0; i < 4; ++i) x.v[4 * c + i] = u[i];
                    if (c == 0) x.vs = *reinterpret_cast<const uint32_t*>(vsp + (chunk >> 2) * 16);
                }
            }
        }
    };

    const uint32_t stride = Split ? kAttWaves : 1;
    AttKV<NB> cur[2], nxt[2];
    uint32_t step = lo + (Split ? wave : 0);
    if (step < end) {
        load(2 * step, cur[0]);
        load(2 * step + 1, cur[1]);
    }
    for (; step < end; step += stride) {
        if (step + stride < end) {
            load(2 * (step + stride), nxt[0]);
            load(2 * (step + stride) + 1, nxt[1]);
        }
        // Scores: tokens 4g + i of both tiles, in powers of two.
        f32x4 s[R][2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
#pragma unroll
            for (int r = 0; r < R; ++r) s[r][x] = zero;
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                const uint32_t b = NB == 8 && j >= 4 ? cur[x].ks >> 8 : cur[x].ks & 0xffu;
                const float sc = __uint_as_float(b << 23);
                const u32x4 kf = {cvt2<0>(cur[x].k[j], sc), cvt2<1>(cur[x].k[j], sc), cvt2<2>(cur[x].k[j], sc),
                                  cvt2<3>(cur[x].k[j], sc)};
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int term = 2; term >= 0; --term) s[r][x] = mfma(kf, qf[r][term][j], s[r][x]);
            }
        }
        const uint32_t at = step * kAttStep;
        // Every row of the wave sees every token of the step: no masks.
        const bool whole = at + kAttStep <= min_limit && cur[0].valid == 16 && cur[1].valid == 16;
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
        // Running maximum, probabilities and their sum; two bf16 terms.
        u32x4 pf[R][2];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float mx = fmaxf(fmaxf(fmaxf(s[r][0][0], s[r][0][1]), fmaxf(s[r][0][2], s[r][0][3])),
                             fmaxf(fmaxf(s[r][1][0], s[r][1][1]), fmaxf(s[r][1][2], s[r][1][3])));
            mx = fmaxf(mx, __shfl_xor(mx, 16, kWave));
            mx = fmaxf(mx, __shfl_xor(mx, 32, kWave));
            if (__any(mx > m[r])) {
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
                    const float p0 = __builtin_amdgcn_exp2f(s[r][x][i] - base);
                    const float p1 = __builtin_amdgcn_exp2f(s[r][x][i + 1] - base);
                    l[r] += p0 + p1;
                    float e0, e1, u0, u1;
                    pf[r][0][2 * x + i / 2] = pack_bf16(p0, p1, &e0, &e1);
                    pf[r][1][2 * x + i / 2] = pack_bf16(e0, e1, &u0, &u1);
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
                const uint32_t code = cur[i >> 2].v[(NB == 8 ? (p >> 2) * 4 : 0) + (i & 3)];
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
                for (int r = 0; r < R; ++r) {
                    o[r][2 * p + h] = mfma(vf, pf[r][1], o[r][2 * p + h]);
                    o[r][2 * p + h] = mfma(vf, pf[r][0], o[r][2 * p + h]);
                }
            }
        }
        // A NaN block of a token that some rows do not see: its 32 dimensions of
        // the rows that do.
        if (!whole && __any(nan_v)) {
            for (uint32_t x = 0; x < 2; ++x) {
                uint32_t valid;
                const uint8_t* base = place(2 * step + x, &valid);
                const uint32_t t0 = (at + 16 * x) & (a.c.page - 1);
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
        cur[0] = nxt[0];
        cur[1] = nxt[1];
    }

#pragma unroll
    for (int r = 0; r < R; ++r) {
        l[r] += __shfl_xor(l[r], 16, kWave);
        l[r] += __shfl_xor(l[r], 32, kWave);
    }
    // Lane (n, g) has dimensions kJ (4g + i) + j of row n in o[.][j][i].
    const uint64_t part0 = (((uint64_t)tile_id * a.c.kv_heads + head) * a.splits + split) * kRows;
    const uint32_t dp = 32 * nb;
    float* const pm = a.part;  // [rows][2] of all, then [rows][dp] of all
    float* const po = a.part + (uint64_t)a.tiles * a.c.kv_heads * a.splits * kRows * 2;
    auto store_row = [&](uint32_t row, float mm, float ll, uint32_t d, const float* v, int count) {
        // `count` values from dimension d of row `row` of the tile, not yet divided
        const uint32_t rr = t.first + row;
        if (rr >= t.rows) return;
        if (a.splits > 1) {
            if (d == 0) {
                pm[(part0 + row) * 2] = mm;
                pm[(part0 + row) * 2 + 1] = ll;
            }
            float* p = po + (part0 + row) * dp + d;
#pragma unroll
            for (int i = 0; i < count; ++i)
                if (d + i < dp) p[i] = v[i];
        } else {
            const float f = ll == 0.0f ? 0.0f : 1.0f / ll;
            float* p = a.out + ((uint64_t)(t.q0 + rr / a.group) * a.q_heads + head * a.group + rr % a.group) * a.dim + d;
#pragma unroll
            for (int i = 0; i < count; ++i)
                if (d + i < a.dim) p[i] = ll == 0.0f ? 0.0f : v[i] * f;
        }
    };
    if constexpr (!Split) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v[kJ];
#pragma unroll
                for (int j = 0; j < kJ; ++j) v[j] = o[r][j][i];
                store_row(wave * 16 * R + 16 * r + n, m[r], l[r], kJ * (4 * g + i), v, kJ);
            }
    } else {
        // Join the waves: to the common maximum, then add.
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
                for (int j = 0; j < kJ; ++j) so[wave][n][kJ * (4 * g + i) + j] = o[r][j][i];
            __syncthreads();
            const uint32_t row = threadIdx.x / 16;
            float mm = ninf, ll = 0.0f, f[kAttWaves];
#pragma unroll
            for (int w = 0; w < kAttWaves; ++w) mm = fmaxf(mm, sm[w][row]);
#pragma unroll
            for (int w = 0; w < kAttWaves; ++w) {
                // a wave that saw nothing holds zeros (or NaN, which stays)
                f[w] = sm[w][row] == ninf ? 1.0f : __builtin_amdgcn_exp2f(sm[w][row] - mm);
                ll += sl[w][row] * f[w];
            }
            for (uint32_t d = (threadIdx.x % 16) * 4; d < (uint32_t)(16 * kJ); d += 64) {
                float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < kAttWaves; ++w) {
                    const f32x4 u = *reinterpret_cast<const f32x4*>(&so[w][row][d]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] += u[i] * f[w];
                }
                store_row(16 * r + row, mm, ll, d, v, 4);
            }
        }
    }
}

// Joins a tile's splits.
template <uint32_t kRows>
__global__ __launch_bounds__(kAttCombine) void att_combine_kernel(AttArgs a) {
    const uint32_t head = blockIdx.y;
    const uint32_t tile_id = a.tile0 + blockIdx.x;
    const AttTile t = att_tile<kRows>(a, tile_id);
    if (!t.ok) return;
    const uint32_t last_row = min(t.first + kRows, t.rows) - 1;
    const uint32_t steps = att_steps(att_limit(a, t, last_row)), share = att_share(steps, a.splits);
    const uint32_t used = steps ? (steps + share - 1) / share : 0;
    const uint64_t part0 = ((uint64_t)tile_id * a.c.kv_heads + head) * a.splits * kRows;
    const float* pm = a.part;
    const float* po = a.part + (uint64_t)a.tiles * a.c.kv_heads * a.splits * kRows * 2;
    const uint32_t dp = 32 * a.c.nb, per_row = dp / 4;
    const float ninf = -__builtin_inff();
    for (uint32_t i = threadIdx.x; i < kRows * per_row; i += kAttCombine) {
        const uint32_t row = i / per_row, d = (i - row * per_row) * 4, rr = t.first + row;
        if (rr >= t.rows) break;
        float mm = ninf, ll = 0.0f;
        for (uint32_t z = 0; z < used; ++z) mm = fmaxf(mm, pm[(part0 + z * kRows + row) * 2]);
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        for (uint32_t z = 0; z < used; ++z) {
            const uint64_t at = part0 + z * kRows + row;
            const float mz = pm[at * 2];
            const float f = mz == ninf ? 1.0f : __builtin_amdgcn_exp2f(mz - mm);
            ll += pm[at * 2 + 1] * f;
            v += *reinterpret_cast<const f32x4*>(po + at * dp + d) * f;
        }
        float* p = a.out + ((uint64_t)(t.q0 + rr / a.group) * a.q_heads + head * a.group + rr % a.group) * a.dim;
        const float f = 1.0f / ll;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (d + k < a.dim) p[d + k] = ll == 0.0f ? 0.0f : v[k] * f;
    }
}

struct AttPlan {
    uint32_t rows;  // rows of a workgroup's tile
    uint32_t tiles, splits;
    uint64_t bytes;  // workspace
};

static int att_plan(uint64_t num_seqs, uint64_t tokens, uint64_t q_heads, uint64_t kv_heads, uint64_t page_size,
                    uint64_t max_pages, uint32_t nb, AttPlan* p) {
    const uint64_t group = q_heads / kv_heads;
    p->rows = 16;
    const uint64_t tiles = tokens * group / p->rows + num_seqs;
    if (tiles > 0x3fffffull) return KORE_HIP_ERR_OVERFLOW;
    p->tiles = (uint32_t)tiles;
    const uint64_t busy = std::max<uint64_t>(1, std::max(std::min(num_seqs, tokens), tokens * group / p->rows)) * kv_heads;
    const uint64_t cap = std::max<uint64_t>(1, max_pages * page_size / 256);
    p->splits = (uint32_t)std::min<uint64_t>({(512 + busy - 1) / busy, cap, 1024});
    p->bytes = p->splits > 1 ? tiles * kv_heads * p->splits * p->rows * (2 + 32ull * nb) * 4 : 0;
    return KORE_HIP_OK;
}

static int att_check(uint64_t num_seqs, uint64_t tokens, uint64_t q_heads, uint64_t kv_heads, uint64_t head_dim,
                     uint64_t num_pages, uint64_t page_size, uint64_t max_pages, Q4Cache* c, AttPlan* p,
                     uint64_t* bytes) {
    const int st = q4_layout(num_pages, page_size, kv_heads, head_dim, c, bytes);
    if (st != KORE_HIP_OK) return st;
    if (kv_heads == 0 || q_heads % kv_heads) return KORE_HIP_ERR_BAD_DIM;
    if (num_seqs > 0x7fffffffull || tokens > 0x7fffffffull || q_heads > 65535u ||
        max_pages > 0xffffffffull / page_size || (num_seqs && max_pages > kMaxElements / num_seqs) ||
        tokens * q_heads > 0xffffffffull)
        return KORE_HIP_ERR_OVERFLOW;
    return att_plan(num_seqs, tokens, q_heads, kv_heads, page_size, max_pages, c->nb, p);
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
    a.tiles = p.tiles;
    a.splits = p.splits;
    a.scale_log2 = (float)((double)scale * 1.4426950408889634);
    a.causal = causal != 0;
    hipStream_t s = (hipStream_t)stream;
    // A launch holds fewer than 2^32 threads: tiles in bands.
    const uint32_t band = (uint32_t)std::max<uint64_t>(1, 0x400000u / (kv_heads * p.splits));
    for (a.tile0 = 0; a.tile0 < p.tiles; a.tile0 += band) {
        const dim3 grid(std::min(band, p.tiles - a.tile0), (uint32_t)kv_heads, p.splits), block(kAttBlock);
        if (a.c.nb <= 2) hipLaunchKernelGGL((att_kernel<2, 1, true>), grid, block, 0, s, a);
        else if (a.c.nb <= 4) hipLaunchKernelGGL((att_kernel<4, 1, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((att_kernel<8, 1, true>), grid, block, 0, s, a);
        const int rc = launch_status();
        if (rc != KORE_HIP_OK) return rc;
    }
    if (p.splits == 1) return KORE_HIP_OK;
    for (a.tile0 = 0; a.tile0 < p.tiles; a.tile0 += band) {
        const dim3 grid(std::min(band, p.tiles - a.tile0), (uint32_t)kv_heads);
        hipLaunchKernelGGL(att_combine_kernel<16>, grid, dim3(kAttCombine), 0, s, a);
        const int rc = launch_status();
        if (rc != KORE_HIP_OK) return rc;
    }
    return KORE_HIP_OK;
}
