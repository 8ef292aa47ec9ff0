// qk_norm_rope.hip -- RMSNorm of every query and key head with the rotary
// embedding in the same pass, and its backward.
//
// Per row x (one head of one token, D values), weight w, position p:
//   n = x / sqrt(mean(x^2) + eps)          (per head, over D)
//   y = R(p) (n * w)                        pairs (i, i + D/2) or (2i, 2i + 1)
//   R(p): (a, b) -> (a cos - b sin, a sin + b cos), angle = p * inv_freq[i]
// Backward, for dy:  g = R(p)^T dy,  u = g * w,
//   dw = sum over rows of g * n,   dx = inv * (u - n * mean(u * n)).
//
// Angles: p * inv_freq is formed and reduced to a part of a turn in f64 (the
// product of a 32-bit position and a 24-bit table entry needs 56 bits; in f32
// the angle of position 100,000 would be off by up to 0.004 rad), then sincospi
// in f32.  Sums of squares and the weight gradients are f32 trees.
//
// Bound: HBM, 8 bytes a value forward (12 backward).  A row lies in a group of
// lanes (D/8 of them, rounded up to a power of two); a lane holds the four
// floats at 4l and the four at D/2 + 4l, so a half-split pair never leaves its
// lane and the row's sums are all that crosses lanes.
//
// 8 x 2048 tokens, 32 + 8 heads of 128: forward 671 MB in 105 us (6.4 TB/s), backward
// 1007 MB in 165 us (6.1 TB/s) and 4.5 for dw (a copy of 2 GiB moves 4.5 TB/s, one
// that the last cache holds 8.2).  One token 3.0 us, which is the launch.
#include <algorithm>
#include <initializer_list>

#include "common.hpp"
#include "kore_hip_internal.hpp"

namespace kore {

constexpr uint32_t kQkMaxHeadDim = 1024;
constexpr uint32_t kQkVecHeadDim = 512;  // 64 lanes a row
constexpr int kQkBlock = 128;
constexpr int kQkBwBlock = 256;
constexpr uint32_t kQkBwParts = 1024;   // partial dw rows at most

struct QkArgs {
    const float* x[2];   // q, k
    const float* dy[2];  // backward: gradients of the outputs
    float* y[2];         // outputs (forward) or gradients of q, k (backward)
    const float* w[2];
    const float* inv_freq;
    const uint32_t* positions;  // or null: start_pos + token % seq_len
    float* part;                // backward: [parts[0] of q, then parts[1] of k][D]
    uint64_t xs[2], dys[2], ys[2];  // floats between two tokens
    uint64_t tokens, token0, seq_len, start_pos;
    uint32_t heads[2];
    uint32_t dim;
    uint32_t chunks[2];  // forward: workgroups of a token's q and k rows
    uint32_t parts[2];   // backward: workgroups of q, of k
    uint32_t span;       // backward: tokens that a workgroup's rows may touch
    float eps;
};

__device__ __forceinline__ uint64_t qk_position(const QkArgs& a, uint64_t token) {
    return a.positions ? (uint64_t)a.positions[token] : a.start_pos + (a.token0 + token) % a.seq_len;
}

__device__ __forceinline__ float2 qk_cos_sin(uint64_t pos, float inv_freq) {
    double t = (double)pos * (double)inv_freq * 0.15915494309189533577;  // turns
    t -= rint(t);
    float s, c;
    sincospif((float)(t + t), &s, &c);
    return make_float2(c, s);
}

template <int kCtrl>
__device__ __forceinline__ float dpp_mov(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), kCtrl, 0xf, 0xf, true));
}

// Sum over the N lanes of a group (a power of two, aligned), in every lane.
template <int N>
__device__ __forceinline__ float group_sum(float v) {
    if (N >= 2) v += dpp_mov<0xb1>(v);   // quad_perm 1,0,3,2
    if (N >= 4) v += dpp_mov<0x4e>(v);   // quad_perm 2,3,0,1
    if (N >= 8) v += dpp_mov<0x141>(v);  // row_half_mirror
    if (N >= 16) v += dpp_mov<0x140>(v);  // row_mirror
    if (N >= 32) v += __shfl_xor(v, 16, kWave);
    if (N >= 64) v += __shfl_xor(v, 32, kWave);
    return v;
}

// Rows are read past the caches (kPast) only where they do not fit the last one (256
// MB): up to 184 MB in and out the caches give 10 % (backward, 4000 x 24 heads of 96:
// 23.3 -> 20.7 us; forward, 4096 x 40 heads of 128: 28.4 -> 25.4), at 336 MB they cost
// 4 % (54.0 -> 56.4), at 1007 MB 8 % (171 -> 184).  Results always go past them (through
// them 12.3 us where 11.2).
constexpr uint64_t kQkCached = 192ull << 20;

template <bool kPast>
__device__ __forceinline__ f32x4 ld4(const float* p) {
    const f32x4_a4* q = reinterpret_cast<const f32x4_a4*>(p);
    if constexpr (kPast) return (f32x4)__builtin_nontemporal_load(q);
    return (f32x4)*q;
}
__device__ __forceinline__ f32x4 ld4_cached(const float* p) { return ld4<false>(p); }
__device__ __forceinline__ void st4(float* p, f32x4 v) { __builtin_nontemporal_store((f32x4_a4)v, reinterpret_cast<f32x4_a4*>(p)); }

// The lane's four (cos, sin): half-split pairs 4l .. 4l + 3; interleaved
// 2l, 2l + 1 (its first float4) and D/4 + 2l, D/4 + 2l + 1 (its second).
template <bool Interleaved>
__device__ __forceinline__ void lane_cs(const float2* cs, uint32_t l, uint32_t dim, float2 o[4]) {
    const uint32_t a = Interleaved ? 2 * l : 4 * l, b = Interleaved ? dim / 4 + 2 * l : 4 * l + 2;
    o[0] = cs[a];
    o[1] = cs[a + 1];
    o[2] = cs[b];
    o[3] = cs[b + 1];
}

// Rotates the lane's eight values; Back: by the negative angle.
template <bool Interleaved, bool Back>
__device__ __forceinline__ void lane_rotate(f32x4& a, f32x4& b, const float2 cs[4]) {
    float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int j0 = Interleaved ? 2 * i : i, j1 = Interleaved ? 2 * i + 1 : i + 4;
        const float c = cs[i].x, s = Back ? -cs[i].y : cs[i].y;
        const float v0 = v[j0], v1 = v[j1];
        v[j0] = __builtin_fmaf(v0, c, -(v1 * s));
        v[j1] = __builtin_fmaf(v0, s, v1 * c);
    }
    a = {v[0], v[1], v[2], v[3]};
    b = {v[4], v[5], v[6], v[7]};
}

__device__ __forceinline__ float dot4(f32x4 a, f32x4 b) {
    return __builtin_fmaf(a.x, b.x, __builtin_fmaf(a.y, b.y, __builtin_fmaf(a.z, b.z, a.w * b.w)));
}

// One workgroup: 128 / LPR rows of one token's Q or K.  The row's loads are
// issued first; the token's cos/sin are computed while they are in flight.
template <int LPR, bool Interleaved, bool kPast>
__global__ __launch_bounds__(kQkBlock) void qk_norm_rope_kernel(QkArgs a) {
    constexpr int kRows = kQkBlock / LPR;
    __shared__ float2 cs[LPR * 4];
    const uint32_t per_token = a.chunks[0] + a.chunks[1];
    const uint64_t token = blockIdx.x / per_token;
    const uint32_t chunk = blockIdx.x % per_token;
    const int t = chunk >= a.chunks[0];
    const uint32_t row = (t ? chunk - a.chunks[0] : chunk) * kRows + threadIdx.x / LPR;
    const uint32_t l = threadIdx.x % LPR, half = a.dim >> 1;
    const bool ok = row < a.heads[t] && l < a.dim >> 3;
    f32x4 x0 = {0.f, 0.f, 0.f, 0.f}, x1 = x0, w0 = x0, w1 = x0;
    if (ok) {
        const float* p = a.x[t] + token * a.xs[t] + (uint64_t)row * a.dim + 4 * l;
        x0 = ld4<kPast>(p);
        x1 = ld4<kPast>(p + half);
        w0 = ld4_cached(a.w[t] + 4 * l);
        w1 = ld4_cached(a.w[t] + half + 4 * l);
    }
    const uint64_t pos = qk_position(a, token);
    for (uint32_t i = threadIdx.x; i < half; i += kQkBlock) cs[i] = qk_cos_sin(pos, a.inv_freq[i]);
    __syncthreads();
    const float ss = group_sum<LPR>(dot4(x0, x0) + dot4(x1, x1));
    if (!ok) return;
    const float inv = 1.0f / sqrtf(ss / (float)a.dim + a.eps);
    f32x4 y0 = x0 * inv * w0, y1 = x1 * inv * w1;
    float2 c[4];
    lane_cs<Interleaved>(cs, l, a.dim, c);
    lane_rotate<Interleaved, false>(y0, y1, c);
    float* o = a.y[t] + token * a.ys[t] + (uint64_t)row * a.dim + 4 * l;
    st4(o, y0);
    st4(o + half, y1);
}

// Any even D: one wave a row, a lane takes the pairs lane, lane + 64, ...
template <bool Interleaved>
__global__ __launch_bounds__(kQkBwBlock) void qk_norm_rope_any_kernel(QkArgs a) {
    const uint64_t r = (uint64_t)blockIdx.x * (kQkBwBlock / kWave) + threadIdx.x / kWave;
    const uint32_t heads = a.heads[0] + a.heads[1], half = a.dim >> 1;
    const uint64_t token = r / heads;
    if (token >= a.tokens) return;
    uint32_t row = (uint32_t)(r - token * heads);
    const int t = row >= a.heads[0];
    if (t) row -= a.heads[0];
    const float* x = a.x[t] + token * a.xs[t] + (uint64_t)row * a.dim;
    float* y = a.y[t] + token * a.ys[t] + (uint64_t)row * a.dim;
    float ss = 0.0f;
    for (uint32_t i = lane_id(); i < a.dim; i += kWave) ss = __builtin_fmaf(x[i], x[i], ss);
    const float inv = 1.0f / sqrtf(group_sum<kWave>(ss) / (float)a.dim + a.eps);
    const uint64_t pos = qk_position(a, token);
    for (uint32_t i = lane_id(); i < half; i += kWave) {
        const uint32_t j0 = Interleaved ? 2 * i : i, j1 = Interleaved ? 2 * i + 1 : i + half;
        const float2 c = qk_cos_sin(pos, a.inv_freq[i]);
        const float v0 = x[j0] * inv * a.w[t][j0], v1 = x[j1] * inv * a.w[t][j1];
        y[j0] = __builtin_fmaf(v0, c.x, -(v1 * c.y));
        y[j1] = __builtin_fmaf(v0, c.y, v1 * c.x);
    }
}

// Backward: the rows of Q (or of K), [tokens][heads], are dealt out in runs of one
// row a lane group, so that the grid sweeps one contiguous band at a time (a
// workgroup with a run of its own measured 186-205 us where this takes 166).  A
// run's loads are in flight while the one before it is worked on, and its tokens'
// cos/sin are computed for it meanwhile.  Each lane keeps the dw of its eight
// dimensions over all its rows; the groups' sums meet in LDS at the end and leave as
// one partial row a workgroup.  Whole: all lanes of a group hold values (D = 8 LPR).
template <int LPR, bool Interleaved, bool Whole, bool kPast>
__global__ __launch_bounds__(kQkBwBlock) void qk_norm_rope_bwd_kernel(QkArgs a) {
    constexpr uint32_t kGroups = kQkBwBlock / LPR;
    extern __shared__ f32x4 qk_lds[];  // cos/sin [2][span][D / 2], later sums [groups][D]
    float2* cs = reinterpret_cast<float2*>(qk_lds);
    float* red = reinterpret_cast<float*>(qk_lds);
    const uint32_t lane = threadIdx.x % LPR, group = threadIdx.x / LPR, half = a.dim >> 1;
    const bool ok = Whole || lane < a.dim >> 3;
    const uint32_t l = Whole ? lane : min(lane, (a.dim >> 3) - 1);
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    const int t = blockIdx.x >= a.parts[0];
    const uint32_t block = t ? blockIdx.x - a.parts[0] : blockIdx.x;
    const uint32_t heads = a.heads[t], stride = a.parts[t] * kGroups, rows = (uint32_t)a.tokens * heads;
    const float* const x = a.x[t];
    const float* const dy = a.dy[t];
    float* const y = a.y[t];
    const uint64_t xs = a.xs[t], dys = a.dys[t], ys = a.ys[t];
    const f32x4 w0 = ok ? ld4_cached(a.w[t] + 4 * l) : zero, w1 = ok ? ld4_cached(a.w[t] + half + 4 * l) : zero;
    const float inv_dim = 1.0f / (float)a.dim;
    f32x4 acc0 = zero, acc1 = zero;
    auto load = [&](uint32_t run, f32x4 (&o)[4]) {
        const uint32_t r = min(run + group, rows - 1);  // past the end: a row that is not used
        const uint32_t tok = r / heads, row = r - tok * heads;
        const float* p = x + tok * xs + (uint64_t)row * a.dim + 4 * l;
        const float* d = dy + tok * dys + (uint64_t)row * a.dim + 4 * l;
        o[0] = ld4<kPast>(p);
        o[1] = ld4<kPast>(p + half);
        o[2] = ld4<kPast>(d);
        o[3] = ld4<kPast>(d + half);
    };
    auto angles = [&](uint32_t run, float2* to) {
        if (run >= rows) return;
        const uint32_t first = run / heads, n = (min(run + kGroups, rows) - 1) / heads - first + 1;
        for (uint32_t i = threadIdx.x; i < n * half; i += kQkBwBlock) {
            const uint32_t tok = i / half, j = i - tok * half;
            to[i] = qk_cos_sin(qk_position(a, first + tok), a.inv_freq[j]);
        }
    };
    auto work = [&](uint32_t run, const f32x4 (&v)[4], const float2* from) {
        const uint32_t r = run + group;
        if (r >= rows) return;
        const uint32_t tok = r / heads, row = r - tok * heads;
        float2 c[4];
        lane_cs<Interleaved>(from + (tok - run / heads) * half, l, a.dim, c);
        const f32x4 x0 = ok ? v[0] : zero, x1 = ok ? v[1] : zero;
        f32x4 g0 = ok ? v[2] : zero, g1 = ok ? v[3] : zero;
        lane_rotate<Interleaved, true>(g0, g1, c);
        const f32x4 u0 = g0 * w0, u1 = g1 * w1;
        const float ss = group_sum<LPR>(dot4(x0, x0) + dot4(x1, x1));
        const float ux = group_sum<LPR>(dot4(u0, x0) + dot4(u1, x1));
        const float inv = 1.0f / sqrtf(ss / (float)a.dim + a.eps);
        const f32x4 n0 = x0 * inv, n1 = x1 * inv;
        acc0 += g0 * n0;
        acc1 += g1 * n1;
        const float mean = ux * inv * inv_dim;
        if (ok) {
            float* o = y + tok * ys + (uint64_t)row * a.dim + 4 * l;
            st4(o, (u0 - n0 * mean) * inv);
            st4(o + half, (u1 - n1 * mean) * inv);
        }
    };
    f32x4 v[2][4];
    uint32_t run = block * kGroups;
    load(run, v[0]);
    angles(run, cs);
    __syncthreads();
    for (; run < rows; run += 2 * stride) {
        load(run + stride, v[1]);
        angles(run + stride, cs + a.span * half);
        work(run, v[0], cs);
        __syncthreads();
        if (run + stride >= rows) break;
        load(run + 2 * stride, v[0]);
        angles(run + 2 * stride, cs);
        work(run + stride, v[1], cs + a.span * half);
        __syncthreads();
    }
    __syncthreads();
    if (ok) {
        float* o = red + group * a.dim;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            o[4 * l + j] = acc0[j];
            o[half + 4 * l + j] = acc1[j];
        }
    }
    __syncthreads();
    for (uint32_t d = threadIdx.x; d < a.dim; d += kQkBwBlock) {
        float s = 0.0f;
        for (uint32_t g = 0; g < kGroups; ++g) s += red[g * a.dim + d];
        a.part[(uint64_t)blockIdx.x * a.dim + d] = s;
    }
}

// Backward, any even D: one wave a row; each wave adds its rows' dw to a row of
// its own in LDS (a lane touches only its pairs).
template <bool Interleaved>
__global__ __launch_bounds__(kQkBwBlock) void qk_norm_rope_bwd_any_kernel(QkArgs a) {
    constexpr uint32_t kWaves = kQkBwBlock / kWave;
    extern __shared__ f32x4 qk_lds[];
    float* dw = reinterpret_cast<float*>(qk_lds);  // [kWaves][D]
    const uint32_t wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, half = a.dim >> 1;
    const int t = blockIdx.x >= a.parts[0];
    const uint32_t block = t ? blockIdx.x - a.parts[0] : blockIdx.x;
    const uint32_t heads = a.heads[t], rows = (uint32_t)a.tokens * heads;
    for (uint32_t i = threadIdx.x; i < kWaves * a.dim; i += kQkBwBlock) dw[i] = 0.0f;
    __syncthreads();
    float* mine = dw + wave * a.dim;
    const float* w = a.w[t];
    for (uint32_t r = block * kWaves + wave; r < rows; r += a.parts[t] * kWaves) {
        const uint32_t token = r / heads, row = r - token * heads;
        const float* x = a.x[t] + token * a.xs[t] + (uint64_t)row * a.dim;
        const float* dy = a.dy[t] + token * a.dys[t] + (uint64_t)row * a.dim;
        float* y = a.y[t] + token * a.ys[t] + (uint64_t)row * a.dim;
        const uint64_t pos = qk_position(a, token);
        float ss = 0.0f, ux = 0.0f;
        for (uint32_t i = lane; i < half; i += kWave) {
            const uint32_t j0 = Interleaved ? 2 * i : i, j1 = Interleaved ? 2 * i + 1 : i + half;
            const float2 c = qk_cos_sin(pos, a.inv_freq[i]);
            const float g0 = __builtin_fmaf(dy[j0], c.x, dy[j1] * c.y), g1 = __builtin_fmaf(dy[j1], c.x, -(dy[j0] * c.y));
            ss += __builtin_fmaf(x[j0], x[j0], x[j1] * x[j1]);
            ux += __builtin_fmaf(g0 * w[j0], x[j0], g1 * w[j1] * x[j1]);
        }
        ss = group_sum<kWave>(ss);
        ux = group_sum<kWave>(ux);
        const float inv = 1.0f / sqrtf(ss / (float)a.dim + a.eps);
        const float mean = ux * inv / (float)a.dim;
        for (uint32_t i = lane; i < half; i += kWave) {
            const uint32_t j0 = Interleaved ? 2 * i : i, j1 = Interleaved ? 2 * i + 1 : i + half;
            const float2 c = qk_cos_sin(pos, a.inv_freq[i]);
            const float g0 = __builtin_fmaf(dy[j0], c.x, dy[j1] * c.y), g1 = __builtin_fmaf(dy[j1], c.x, -(dy[j0] * c.y));
            const float n0 = x[j0] * inv, n1 = x[j1] * inv;
            mine[j0] += g0 * n0;
            mine[j1] += g1 * n1;
            y[j0] = (g0 * w[j0] - n0 * mean) * inv;
            y[j1] = (g1 * w[j1] - n1 * mean) * inv;
        }
    }
    __syncthreads();
    for (uint32_t d = threadIdx.x; d < a.dim; d += kQkBwBlock) {
        float s = 0.0f;
        for (uint32_t v = 0; v < kWaves; ++v) s += dw[v * a.dim + d];
        a.part[(uint64_t)blockIdx.x * a.dim + d] = s;
    }
}

// dw[t][d] = the partial rows' sum, in a fixed order: 64 row slots a column, eight
// rows of a slot in flight.
constexpr int kQkRedCols = 16, kQkRedSlots = 64, kQkRedFlight = 8;
__global__ __launch_bounds__(kQkRedCols* kQkRedSlots) void qk_norm_rope_dw_kernel(const float* part, uint32_t q_parts,
                                                                                  uint32_t k_parts, uint32_t dim,
                                                                                  float* dqw, float* dkw) {
    __shared__ float red[kQkRedSlots][kQkRedCols + 1];
    const uint32_t c = threadIdx.x % kQkRedCols, slot = threadIdx.x / kQkRedCols;
    const uint32_t col = blockIdx.x * kQkRedCols + c;
    const int t = blockIdx.y;  // 0: q, 1: k
    const uint32_t parts = t ? k_parts : q_parts;
    if (t) part += (uint64_t)q_parts * dim;
    float s = 0.0f;
    if (col < dim) {
        for (uint32_t p = slot; p < parts; p += kQkRedSlots * kQkRedFlight) {
            float v[kQkRedFlight];
#pragma unroll
            for (int i = 0; i < kQkRedFlight; ++i) {
                const uint32_t at = p + i * kQkRedSlots;
                v[i] = at < parts ? part[(uint64_t)at * dim + col] : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < kQkRedFlight; ++i) s += v[i];
        }
    }
    red[slot][c] = s;
    __syncthreads();
#pragma unroll
    for (int n = kQkRedSlots / 2; n >= 1; n /= 2) {
        if (slot < (uint32_t)n) red[slot][c] += red[slot + n][c];
        __syncthreads();
    }
    float* o = t ? dkw : dqw;
    if (slot == 0 && col < dim && o) o[col] = red[0][c];
}

// Whether rows of `wa` floats every `sa` from a meet rows of `wb` every `sb`
// from b, n of each.  Rows of one stride may lie between each other.
static bool rows_overlap(const float* a, uint64_t sa, uint64_t wa, const float* b, uint64_t sb, uint64_t wb,
                         uint64_t n) {
    if (!a || !b || !wa || !wb || !n) return false;
    const uintptr_t p = (uintptr_t)a, q = (uintptr_t)b;
    if (!(p < q + ((n - 1) * sb + wb) * 4 && q < p + ((n - 1) * sa + wa) * 4)) return false;
    if (sa != sb || n == 1 || ((q - p) & 3)) return true;
    const uint64_t off = q >= p ? (q - p) / 4 % sa : (sa - (p - q) / 4 % sa) % sa;
    return off < wa || off + wb > sa;
}

static uint32_t qk_lanes(uint32_t dim) {
    uint32_t l = 1;
    while (l * 8 < dim) l *= 2;
    return l;
}

static bool qk_vector(uint32_t dim) { return dim % 8 == 0 && dim <= kQkVecHeadDim; }

struct QkPlan {
    uint32_t parts[2];  // workgroups of q and k, each a partial dw row
    uint32_t groups;    // rows of a run
};

// 1024 workgroups, four to a CU, shared out as Q's and K's heads are.
static QkPlan qk_plan(uint64_t tokens, uint32_t q_heads, uint32_t k_heads, uint32_t dim) {
    QkPlan p = {};
    p.groups = kQkBwBlock / (qk_vector(dim) ? qk_lanes(dim) : kWave);
    const uint32_t heads[2] = {q_heads, k_heads};
    for (int t = 0; t < 2; ++t) {
        const uint64_t share = (uint64_t)kQkBwParts * heads[t] / ((uint64_t)q_heads + k_heads);
        p.parts[t] = (uint32_t)std::min((tokens * heads[t] + p.groups - 1) / p.groups, std::max<uint64_t>(share, 1));
    }
    return p;
}

// Checks shared by both directions; fills dims, strides and the launch's tokens.
static int qk_check(QkArgs* a, uint64_t batch, uint64_t seq_len, uint32_t q_heads, uint32_t k_heads, uint32_t dim,
                    uint64_t start_pos, const uint32_t* positions) {
    if ((dim & 1u) || dim > kQkMaxHeadDim) return KORE_HIP_ERR_BAD_DIM;
    if (q_heads > 65535u || k_heads > 65535u || a->tokens > 0x7fffffffull) return KORE_HIP_ERR_OVERFLOW;
    if (!positions && start_pos + seq_len < start_pos) return KORE_HIP_ERR_OVERFLOW;
    a->heads[0] = q_heads;
    a->heads[1] = k_heads;
    a->dim = dim;
    a->seq_len = seq_len;
    a->start_pos = start_pos;
    a->positions = positions;
    for (int t = 0; t < 2; ++t) {
        const uint64_t row = (uint64_t)a->heads[t] * dim;
        for (uint64_t* s : {&a->xs[t], &a->dys[t], &a->ys[t]}) {
            if (*s == 0) *s = row;
            if (*s < row) return KORE_HIP_ERR_BAD_DIM;
            uint64_t span;
            if (!mul_ok(a->tokens, *s, &span) || span > kMaxElements) return KORE_HIP_ERR_OVERFLOW;
        }
    }
    return KORE_HIP_OK;
}

// An output may be one of its inputs (the same rows) or apart from all inputs
// and from the other output.
static bool qk_alias(const QkArgs& a, const float* const in[2], const uint64_t is[2], bool own_ok) {
    for (int t = 0; t < 2; ++t)
        for (int u = 0; u < 2; ++u) {
            if (!a.heads[t] || !a.heads[u]) continue;
            if (own_ok && t == u && a.y[t] == in[u] && a.ys[t] == is[u]) continue;
            if (rows_overlap(a.y[t], a.ys[t], (uint64_t)a.heads[t] * a.dim, in[u], is[u],
                             (uint64_t)a.heads[u] * a.dim, a.tokens))
                return true;
        }
    return false;
}

static bool qk_outputs_alias(const QkArgs& a) {
    return a.heads[0] && a.heads[1] &&
           rows_overlap(a.y[0], a.ys[0], (uint64_t)a.heads[0] * a.dim, a.y[1], a.ys[1],
                        (uint64_t)a.heads[1] * a.dim, a.tokens);
}

// Whether rows of a strided output meet `bytes` bytes at p.
static bool qk_rows_meet(const float* y, uint64_t stride, uint64_t width, uint64_t n, const void* p, uint64_t bytes) {
    if (!y || !p || !n || !width || !bytes) return false;
    const uint64_t lo = (uint64_t)(uintptr_t)p, hi = lo + bytes, at = (uint64_t)(uintptr_t)y;
    const uint64_t first = lo < at ? 0 : std::min((lo - at) / (stride * 4), n - 1);
    for (uint64_t r = first; r < std::min(first + 2, n); ++r)
        if (at + r * stride * 4 < hi && lo < at + (r * stride + width) * 4) return true;
    return false;
}

struct QkFlat {
    const void* p;
    uint64_t bytes;
};

// Whether an output's rows meet what all rows read (weights, table, positions) or
// one of `more`.
static bool qk_meets(const QkArgs& a, std::initializer_list<QkFlat> more) {
    const uint64_t row = (uint64_t)a.dim * 4;
    for (int t = 0; t < 2; ++t) {
        const uint64_t width = (uint64_t)a.heads[t] * a.dim;
        auto meets = [&](const void* p, uint64_t bytes) {
            return qk_rows_meet(a.y[t], a.ys[t], width, a.tokens, p, bytes);
        };
        if (meets(a.w[0], row) || meets(a.w[1], row) || meets(a.inv_freq, row / 2) || meets(a.positions, a.tokens * 4))
            return true;
        for (const QkFlat& f : more)
            if (meets(f.p, f.bytes)) return true;
    }
    return false;
}

#define QK_LANES(L, CALL)                  \
    switch (L) {                           \
        case 1: { CALL(1); } break;        \
        case 2: { CALL(2); } break;        \
        case 4: { CALL(4); } break;        \
        case 8: { CALL(8); } break;        \
        case 16: { CALL(16); } break;      \
        case 32: { CALL(32); } break;      \
        default: { CALL(64); } break;      \
    }

}  // namespace kore

using namespace kore;

extern "C" int kore_hip_qk_norm_rope_f32(const float* q, const float* k, const float* q_weight, const float* k_weight,
                                         const float* inv_freq, const uint32_t* positions, float* q_out, float* k_out,
                                         uint64_t batch, uint64_t seq_len, uint32_t q_heads, uint32_t k_heads,
                                         uint32_t head_dim, uint64_t q_stride, uint64_t k_stride,
                                         uint64_t q_out_stride, uint64_t k_out_stride, uint64_t start_pos, float eps,
                                         int interleaved, kore_stream_t stream) {
    QkArgs a = {};
    if (!mul_ok(batch, seq_len, &a.tokens)) return KORE_HIP_ERR_OVERFLOW;
    if (a.tokens == 0 || head_dim == 0 || (q_heads == 0 && k_heads == 0)) return KORE_HIP_OK;
    a.xs[0] = q_stride;
    a.xs[1] = k_stride;
    a.ys[0] = q_out_stride;
    a.ys[1] = k_out_stride;
    const int st = qk_check(&a, batch, seq_len, q_heads, k_heads, head_dim, start_pos, positions);
    if (st != KORE_HIP_OK) return st;
    if (!inv_freq || (q_heads && (!q || !q_weight || !q_out)) || (k_heads && (!k || !k_weight || !k_out)))
        return KORE_HIP_ERR_NULL_PTR;
    a.x[0] = q;
    a.x[1] = k;
    a.y[0] = q_out;
    a.y[1] = k_out;
    a.w[0] = q_weight;
    a.w[1] = k_weight;
    a.inv_freq = inv_freq;
    a.eps = eps;
    if (qk_alias(a, a.x, a.xs, true) || qk_outputs_alias(a) || qk_meets(a, {})) return KORE_HIP_ERR_ALIAS;
    hipStream_t s = (hipStream_t)stream;
    const bool vec = qk_vector(head_dim);
    const bool past = a.tokens * ((uint64_t)q_heads + k_heads) * head_dim * 8 > kQkCached;
    const uint32_t lanes = qk_lanes(head_dim), rows = kQkBlock / std::min(lanes, 64u);
    a.chunks[0] = (q_heads + rows - 1) / rows;
    a.chunks[1] = (k_heads + rows - 1) / rows;
    // A launch holds fewer than 2^32 threads: tokens in bands.
    const uint64_t threads = vec ? (uint64_t)(a.chunks[0] + a.chunks[1]) * kQkBlock : ((uint64_t)q_heads + k_heads) * kWave;
    const uint64_t band = std::max<uint64_t>(1, 0x40000000ull / threads), all = a.tokens;
    for (uint64_t t = 0; t < all; t += band) {
        a.tokens = std::min(band, all - t);
        a.token0 = t;
        if (vec) {
            const dim3 grid((uint32_t)(a.tokens * (a.chunks[0] + a.chunks[1])));
#define QK_CALL(L)                                                                                                     \
    if (interleaved && past) hipLaunchKernelGGL((qk_norm_rope_kernel<L, true, true>), grid, dim3(kQkBlock), 0, s, a);  \
    else if (interleaved) hipLaunchKernelGGL((qk_norm_rope_kernel<L, true, false>), grid, dim3(kQkBlock), 0, s, a);    \
    else if (past) hipLaunchKernelGGL((qk_norm_rope_kernel<L, false, true>), grid, dim3(kQkBlock), 0, s, a);           \
    else hipLaunchKernelGGL((qk_norm_rope_kernel<L, false, false>), grid, dim3(kQkBlock), 0, s, a);
            QK_LANES(lanes, QK_CALL)
#undef QK_CALL
        } else {
            const uint64_t n = a.tokens * ((uint64_t)q_heads + k_heads);
            const dim3 grid((uint32_t)((n + kQkBwBlock / kWave - 1) / (kQkBwBlock / kWave)));
            if (interleaved) hipLaunchKernelGGL(qk_norm_rope_any_kernel<true>, grid, dim3(kQkBwBlock), 0, s, a);
            else hipLaunchKernelGGL(qk_norm_rope_any_kernel<false>, grid, dim3(kQkBwBlock), 0, s, a);
        }
        const int rc = launch_status();
        if (rc != KORE_HIP_OK) return rc;
        for (int u = 0; u < 2; ++u) {
            if (!a.heads[u]) continue;
            a.x[u] += a.tokens * a.xs[u];
            a.y[u] += a.tokens * a.ys[u];
        }
        if (a.positions) a.positions += a.tokens;
    }
    return KORE_HIP_OK;
}

extern "C" uint64_t kore_hip_qk_norm_rope_backward_workspace_bytes(uint64_t tokens, uint32_t q_heads, uint32_t k_heads,
                                                                   uint32_t head_dim) {
    if (tokens == 0 || head_dim == 0 || head_dim > kQkMaxHeadDim || (q_heads == 0 && k_heads == 0)) return 0;
    const QkPlan p = qk_plan(tokens, q_heads, k_heads, head_dim);
    return ((uint64_t)p.parts[0] + p.parts[1]) * head_dim * sizeof(float);
}

extern "C" int kore_hip_qk_norm_rope_backward_f32(
    const float* grad_q_out, const float* grad_k_out, const float* q, const float* k, const float* q_weight,
    const float* k_weight, const float* inv_freq, const uint32_t* positions, float* grad_q, float* grad_k,
    float* grad_q_weight, float* grad_k_weight, float* workspace, uint64_t workspace_bytes, uint64_t batch,
    uint64_t seq_len, uint32_t q_heads, uint32_t k_heads, uint32_t head_dim, uint64_t grad_q_out_stride,
    uint64_t grad_k_out_stride, uint64_t q_stride, uint64_t k_stride, uint64_t grad_q_stride, uint64_t grad_k_stride,
    uint64_t start_pos, float eps, int interleaved, kore_stream_t stream) {
    QkArgs a = {};
    if (!mul_ok(batch, seq_len, &a.tokens)) return KORE_HIP_ERR_OVERFLOW;
    if (head_dim == 0 || (q_heads == 0 && k_heads == 0)) return KORE_HIP_OK;
    a.dys[0] = grad_q_out_stride;
    a.dys[1] = grad_k_out_stride;
    a.xs[0] = q_stride;
    a.xs[1] = k_stride;
    a.ys[0] = grad_q_stride;
    a.ys[1] = grad_k_stride;
    const int st = qk_check(&a, batch, seq_len, q_heads, k_heads, head_dim, start_pos, positions);
    if (st != KORE_HIP_OK) return st;
    if ((q_heads && !grad_q_weight) || (k_heads && !grad_k_weight)) return KORE_HIP_ERR_NULL_PTR;
    // rows are counted in 32 bits, with room for a sweep of the grid
    if (a.tokens * std::max(q_heads, k_heads) > 0xf0000000ull) return KORE_HIP_ERR_OVERFLOW;
    const uint64_t need = kore_hip_qk_norm_rope_backward_workspace_bytes(a.tokens, q_heads, k_heads, head_dim);
    hipStream_t s = (hipStream_t)stream;
    const QkPlan plan = qk_plan(a.tokens, q_heads, k_heads, head_dim);
    if (a.tokens) {
        if (!inv_freq || !workspace || (q_heads && (!grad_q_out || !q || !q_weight || !grad_q)) ||
            (k_heads && (!grad_k_out || !k || !k_weight || !grad_k)))
            return KORE_HIP_ERR_NULL_PTR;
        if (workspace_bytes < need) return KORE_HIP_ERR_BAD_DIM;
        a.dy[0] = grad_q_out;
        a.dy[1] = grad_k_out;
        a.x[0] = q;
        a.x[1] = k;
        a.y[0] = grad_q;
        a.y[1] = grad_k;
        a.w[0] = q_weight;
        a.w[1] = k_weight;
        a.inv_freq = inv_freq;
        a.eps = eps;
        a.part = workspace;
        for (int t = 0; t < 2; ++t) a.parts[t] = plan.parts[t];
        const uint64_t dw = (uint64_t)head_dim * 4;
        if (qk_alias(a, a.x, a.xs, true) || qk_alias(a, a.dy, a.dys, true) || qk_outputs_alias(a) ||
            qk_meets(a, {{workspace, need}, {grad_q_weight, dw}, {grad_k_weight, dw}}))
            return KORE_HIP_ERR_ALIAS;
        const QkFlat flat[] = {{q_weight, dw}, {k_weight, dw}, {inv_freq, dw / 2}, {positions, a.tokens * 4},
                               {grad_q_weight, dw}, {grad_k_weight, dw}};
        for (const QkFlat& f : flat)
            if (qk_rows_meet(workspace, need / 4, need / 4, 1, f.p, f.bytes)) return KORE_HIP_ERR_ALIAS;
        for (int t = 0; t < 2; ++t)
            if (a.heads[t] && (qk_rows_meet(a.x[t], a.xs[t], (uint64_t)a.heads[t] * head_dim, a.tokens, workspace, need) ||
                               qk_rows_meet(a.dy[t], a.dys[t], (uint64_t)a.heads[t] * head_dim, a.tokens, workspace, need)))
                return KORE_HIP_ERR_ALIAS;
        if (q_heads && k_heads && qk_rows_meet(grad_q_weight, head_dim, head_dim, 1, grad_k_weight, dw))
            return KORE_HIP_ERR_ALIAS;
        const dim3 grid(plan.parts[0] + plan.parts[1]), block(kQkBwBlock);
        const bool past = a.tokens * ((uint64_t)q_heads + k_heads) * head_dim * 12 > kQkCached;
        if (qk_vector(head_dim)) {
            const uint32_t lanes = qk_lanes(head_dim);
            const uint32_t fewest = !q_heads ? k_heads : !k_heads ? q_heads : std::min(q_heads, k_heads);
            a.span = (plan.groups - 1) / fewest + 2;
            const size_t lds = (size_t)std::max(2 * a.span, plan.groups) * head_dim * sizeof(float);
            const bool whole = head_dim == 8 * lanes;
#define QK_FORM(L, I, W)                                                                                               \
    if (past) hipLaunchKernelGGL((qk_norm_rope_bwd_kernel<L, I, W, true>), grid, block, lds, s, a);                    \
    else hipLaunchKernelGGL((qk_norm_rope_bwd_kernel<L, I, W, false>), grid, block, lds, s, a);
#define QK_CALL(L)                                                                                                     \
    if (interleaved && whole) { QK_FORM(L, true, true) }                                                               \
    else if (interleaved) { QK_FORM(L, true, false) }                                                                  \
    else if (whole) { QK_FORM(L, false, true) }                                                                        \
    else { QK_FORM(L, false, false) }
            QK_LANES(lanes, QK_CALL)
#undef QK_CALL
#undef QK_FORM
        } else {
            const size_t lds = (size_t)(kQkBwBlock / kWave) * head_dim * sizeof(float);
            if (interleaved) hipLaunchKernelGGL(qk_norm_rope_bwd_any_kernel<true>, grid, block, lds, s, a);
            else hipLaunchKernelGGL(qk_norm_rope_bwd_any_kernel<false>, grid, block, lds, s, a);
        }
        const int rc = launch_status();
        if (rc != KORE_HIP_OK) return rc;
    }
    hipLaunchKernelGGL(qk_norm_rope_dw_kernel, dim3((head_dim + kQkRedCols - 1) / kQkRedCols, 2),
                       dim3(kQkRedCols * kQkRedSlots), 0, s, workspace, plan.parts[0], plan.parts[1], head_dim,
                       q_heads ? grad_q_weight : nullptr, k_heads ? grad_k_weight : nullptr);
    return launch_status();
}
