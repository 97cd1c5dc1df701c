// sgpu_score.hip -- what a host that scores or samples several continuations of one prompt needs
// beside the decode engines' own kernels (gfx950):
//   sgpu_rope_rows_*    rotary positions of rows at positions of their own
//   sgpu_logprobs_*     log probabilities of given tokens, entropy and top alternatives of logits
//   sgpu_attn_prefix_*  attention of a batch whose sequences share a long prefix
// fp16 values here are IEEE ones (infinities, NaN and subnormals as they are), unlike the weight
// codes of the GEMVs.
#include <type_traits>

#include "sgpu_rows.h"

namespace {

// ---- rotary positions ----
constexpr int kRopeTable = 2048;      // (cos, sin) pairs a block holds: its rows by rot / 2

// Rows t of x (H heads of HD values, row stride xs) at position pos0 + (pos ? pos[t] : t), rotated
// into y (row stride ys): pair i of a head by turns[i] per position, pairs (i, i + rot/2) or
// (INTER) (2i, 2i + 1); values past rot pass through.  A block takes tb rows: the angles of its
// rows once into LDS, then every head reads them.  VEC: four values a lane and access (rows 16-byte
// aligned, HD, rot and rot/2 whole quads); otherwise a pair or one value a lane.
// Bound: the rows' way through memory; below some hundred rows the launch.  3001 rows of 16 heads of 64 take
// 5.4 us (24.6 MB, 4.5 TB/s), of 40 heads of 128 with 64 rotated values, into fp16, 16.7 us (92 MB, 5.5 TB/s), one
// row 1.8 us.
template <typename O, bool INTER, bool VEC>
__device__ __forceinline__ void rope_rows(const float* x, long long xs, O* y, long long ys, const int* __restrict__ pos,
                                          int pos0, const double* __restrict__ turns, int rot, float mscale, int T, int H,
                                          int HD, int tb, int same) {
    __shared__ float table[2 * kRopeTable];
    const int tid = threadIdx.x, half = rot / 2;
    // (a long list of rows goes over the grid more than once)
    for (int t0 = blockIdx.x * tb; t0 < T; t0 += gridDim.x * tb) {
        const int n = min(tb, T - t0);
        for (int i = tid; i < n * half; i += 256) {
            const int t = i / half;
            const long long p = (long long)pos0 + (pos ? pos[t0 + t] : t0 + t);
            float s, c;
            sincos_turns((double)p * turns[i - t * half], s, c);
            table[2 * i] = c * mscale;
            table[2 * i + 1] = s * mscale;
        }
        __syncthreads();
        // work items of a head: the rotated ones, then what passes through (nothing where y is x)
        const int w = VEC ? 4 : 1;
        const int per = INTER && VEC ? rot / 4 : half / w, rest = same ? 0 : (HD - rot) / w, items = per + rest;
        for (int i = tid; i < n * H * items; i += 256) {
            const int e = i % items, th = i / items, h = th % H, t = th / H;
            const float* xr = x + (t0 + t) * xs + (long long)h * HD;
            O* yr = y + (t0 + t) * ys + (long long)h * HD;
            const float* tab = table + 2 * t * half;
            if (e >= per) {
                const int d = rot + (e - per) * w;
                if constexpr (VEC) {
                    const sgpu_f32x4 a = *reinterpret_cast<const sgpu_f32x4*>(xr + d);
                    const float v[4] = {a[0], a[1], a[2], a[3]};
                    put4(yr + d, v);
                } else {
                    yr[d] = (O)xr[d];
                }
            } else if constexpr (VEC && INTER) {
                const sgpu_f32x4 a = *reinterpret_cast<const sgpu_f32x4*>(xr + 4 * e);
                const sgpu_f32x4 k = *reinterpret_cast<const sgpu_f32x4*>(tab + 4 * e);
                const float v[4] = {a[0] * k[0] - a[1] * k[1], a[0] * k[1] + a[1] * k[0], a[2] * k[2] - a[3] * k[3],
                                    a[2] * k[3] + a[3] * k[2]};
                put4(yr + 4 * e, v);
            } else if constexpr (VEC) {
                const sgpu_f32x4 a = *reinterpret_cast<const sgpu_f32x4*>(xr + 4 * e);
                const sgpu_f32x4 b = *reinterpret_cast<const sgpu_f32x4*>(xr + half + 4 * e);
                float u[4], v[4];
    #pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float c = tab[2 * (4 * e + j)], s = tab[2 * (4 * e + j) + 1];
                    u[j] = a[j] * c - b[j] * s;
                    v[j] = a[j] * s + b[j] * c;
                }
                put4(yr + 4 * e, u);
                put4(yr + half + 4 * e, v);
            } else {
                const int i0 = INTER ? 2 * e : e, i1 = INTER ? 2 * e + 1 : half + e;
                const float a = xr[i0], b = xr[i1], c = tab[2 * e], s = tab[2 * e + 1];
                yr[i0] = (O)(a * c - b * s);
                yr[i1] = (O)(a * s + b * c);
            }
        }
        __syncthreads();                          // the table is the next rows'
    }
}

// ---- log probabilities ----
// A row's statistics relative to its maximum m: S = sum 2^y, W = sum y 2^y, y = (x - m) log2 e.
struct stats {
    float m, s, w;
};
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

__device__ __forceinline__ void join(stats& a, const stats& b) {
    const float m = fmaxf(a.m, b.m);
    const float da = (a.m - m) * kLog2e, db = (b.m - m) * kLog2e;
    const float ea = __builtin_amdgcn_exp2f(da), eb = __builtin_amdgcn_exp2f(db);
    // a part with no weight left adds nothing (its distance may be infinite)
    const float wa = ea > 0.0f ? ea * __builtin_fmaf(da, a.s, a.w) : 0.0f;
    const float wb = eb > 0.0f ? eb * __builtin_fmaf(db, b.s, b.w) : 0.0f;
    a.s = ea * a.s + eb * b.s;
    a.w = wa + wb;
    a.m = m;
}

// Numbers in their order as whole numbers (-0 as +0), the id below them so that the lowest id is
// first among equals.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __float_as_uint(x == 0.0f ? 0.0f : x);
    return b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k ^ (k >> 31 ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ unsigned long long key_of(float x, int id) {
    return ((unsigned long long)order_of(x) << 32) | (uint32_t)~id;
}

constexpr int kTop = 64;               // the most alternatives of a row: a lane each

// Keys in order across the wave, on the vector ALUs (bitonic networks: 21 exchanges sort 64 keys, 6 merge; ranking by
// counting took 28 + 21 us for 64 alternatives of a row where this takes 12 + 8).
// Lane ^ m's value:
__device__ __forceinline__ uint32_t lane_xor(uint32_t x, int m) {
    auto dpp = [](uint32_t v, auto ctrl) __attribute__((always_inline)) {
        return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, 0xf, 0xf, true);
    };
    const int lane = threadIdx.x & 63;
    if (m == 1) return dpp(x, std::integral_constant<int, 0xB1>());                    // quads 1 0 3 2
    if (m == 2) return dpp(x, std::integral_constant<int, 0x4E>());                    // quads 2 3 0 1
    if (m == 4) return dpp(dpp(x, std::integral_constant<int, 0x141>()), std::integral_constant<int, 0x1B>());     // ^ 7, ^ 3
    if (m == 8) return dpp(x, std::integral_constant<int, 0x128>());                   // rows of 16 turned by 8
    if (m == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
        return lane & 16 ? r[0] : r[1];
    }
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return lane & 32 ? r[0] : r[1];
}
__device__ __forceinline__ unsigned long long exchange(unsigned long long key, int m, bool larger) {
    const unsigned long long o =
        (unsigned long long)lane_xor((uint32_t)(key >> 32), m) << 32 | lane_xor((uint32_t)key, m);
    return (o > key) == larger ? o : key;
}
__device__ __forceinline__ unsigned long long sort_up(unsigned long long key) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int size = 2; size <= 64; size *= 2)
#pragma unroll
        for (int m = size / 2; m > 0; m /= 2) key = exchange(key, m, ((lane & m) != 0) != (size < 64 && (lane & size) != 0));
    return key;
}
// The 64 largest of a falling and a rising sequence, falling.
__device__ __forceinline__ unsigned long long merge_down(unsigned long long down, unsigned long long up) {
    const int lane = threadIdx.x & 63;
    unsigned long long key = up > down ? up : down;
#pragma unroll
    for (int m = 32; m > 0; m /= 2) key = exchange(key, m, (lane & m) == 0);
    return key;
}

// Top alternatives of what one wave sees: `best`, lane i's the i-th best key so far (0 where none), and
// n candidates that beat the k-th, up to 127 of them waiting in LDS.
struct top_list {
    unsigned long long* wait;          // kTop + 64 keys
    int k, n;
    unsigned long long best, kth;
};
__device__ __forceinline__ void top_kth(top_list& l) {
    l.kth = (unsigned long long)(uint32_t)__builtin_amdgcn_readlane((int)(l.best >> 32), l.k - 1) << 32 |
            (uint32_t)__builtin_amdgcn_readlane((int)l.best, l.k - 1);
}
__device__ __forceinline__ void top_flush(top_list& l) {
    if (l.n == 0) return;
    const int lane = threadIdx.x & 63;
    lds_sync();
    if (l.n <= 8) {                    // few: each to its place
        for (int i = 0; i < l.n; i++) {
            const unsigned long long key = l.wait[i];
            const int at = __popcll(__ballot(l.best > key));
            const unsigned long long above =
                (unsigned long long)(uint32_t)__shfl_up((int)(l.best >> 32), 1) << 32 | (uint32_t)__shfl_up((int)l.best, 1);
            l.best = lane < at ? l.best : lane == at ? key : above;
        }
        l.n = 0;
    } else {
        const unsigned long long key = lane < l.n ? l.wait[lane] : 0, rest = l.wait[64 + lane];
        lds_sync();
        l.wait[lane] = rest;
        l.n = max(l.n - 64, 0);
        l.best = merge_down(l.best, sort_up(key));
    }
    top_kth(l);
}
__device__ __forceinline__ void top_add(top_list& l, bool in, unsigned long long key) {
    const unsigned long long b = __ballot(in);
    if (!b) return;
    const int lane = threadIdx.x & 63;
    if (in) l.wait[l.n + __popcll(b & ((1ull << lane) - 1))] = key;
    l.n += __popcll(b);
    if (l.n >= 64) top_flush(l);
}
// The largest number of 16 bits, 16 zero bits behind it, that at least k lanes' `order` reaches.
__device__ __forceinline__ uint32_t reached_by(int k, uint32_t order) {
    uint32_t p = 0;
    for (uint32_t bit = 1u << 31; bit >= 1u << 16; bit >>= 1)
        if (__popcll(__ballot(order >= (p | bit))) >= k) p |= bit;
    return p;
}
template <typename X> struct logits;
template <> struct logits<float> {
    typedef sgpu_f32x4 vec;
    __device__ static __forceinline__ vec load(const float* p) { return sgpu_ld4<false>(p); }
};
template <> struct logits<_Float16> {
    typedef f16x8 vec;
    __device__ static __forceinline__ vec load(const _Float16* p) { return *reinterpret_cast<const f16x8_a2*>(p); }
};

constexpr int kLpTile = 32;            // values a lane holds at a time

// Chunk c of row r (V values, C chunks of `len`): its statistics to part[(r * C + c) * 4 ..], its k
// best keys to keys[(r * C + c) * k ..].  256 threads; a wave takes tiles of 64 * kLpTile values.
// One pass: running maximum, sum and weighted sum per lane, joined at the end; a tile's values are summed by themselves,
// in four parts, so that V / 8192 + 10 roundings follow one another, not V / 256.  Bound: fp32, for
// the most part the logits' way through memory (2048 rows of 50257: 79 us, 5.2 TB/s, where the widest reads reach 6.75);
// fp16, the dozen vector instructions and the exponential of each value (1024 rows of 151936: 82 - 89 us, 3.5 - 3.8 TB/s;
// loading a tile ahead made no difference to either).  One row of 151936 is 19 chunks: 3.5 us without alternatives, 6.5 us with 20, 12 us
// with 64, of which the launch is some 2.
template <typename X>
__device__ __forceinline__ void lp_part(const X* __restrict__ x, long long xs, int V, int C, int len, int k,
                                        float* __restrict__ part, unsigned long long* __restrict__ keys) {
    typedef typename logits<X>::vec vec;
    constexpr int VEC = 16 / sizeof(X), NV = kLpTile / VEC;
    __shared__ unsigned long long lists[4][kTop + 64];
    __shared__ stats red[4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = blockIdx.x % C, r = blockIdx.x / C;
    const X* row = x + (long long)r * xs;
    const int v0 = c * len, v1 = min(V, v0 + len);
    top_list top = {lists[wave], k, 0, 0, 0};
    stats a = {-3.402823466e38f, 0.0f, 0.0f};
    for (int t0 = v0 + wave * 64 * kLpTile; t0 < v1; t0 += 4 * 64 * kLpTile) {
        float v[kLpTile];
        if (t0 + 64 * kLpTile <= v1) {
            vec raw[NV];
#pragma unroll
            for (int j = 0; j < NV; j++) raw[j] = logits<X>::load(row + t0 + (j * 64 + lane) * VEC);
#pragma unroll
            for (int j = 0; j < kLpTile; j++) v[j] = (float)raw[j / VEC][j % VEC];
        } else {
#pragma unroll
            for (int j = 0; j < kLpTile; j++) {
                const int i = t0 + ((j / VEC) * 64 + lane) * VEC + j % VEC;
                v[j] = i < v1 ? (float)row[i] : -INFINITY;
            }
        }
        float m = v[0];
#pragma unroll
        for (int j = 1; j < kLpTile; j++) m = fmaxf(m, v[j]);
        const float mn = fmaxf(a.m, m), d = (a.m - mn) * kLog2e, e0 = __builtin_amdgcn_exp2f(d);
        float ts[4] = {0.0f, 0.0f, 0.0f, 0.0f}, tw[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < kLpTile; j++) {
            const float y = (v[j] - mn) * kLog2e, e = __builtin_amdgcn_exp2f(y);
            ts[j % 4] += e;
            tw[j % 4] = __builtin_fmaf(e, fmaxf(y, -256.0f), tw[j % 4]);     // no weight, no part: 0 times an infinity
        }
        const float aw = e0 > 0.0f ? e0 * __builtin_fmaf(d, a.s, a.w) : 0.0f;
        a = {mn, __builtin_fmaf(e0, a.s, (ts[0] + ts[1]) + (ts[2] + ts[3])), aw + ((tw[0] + tw[1]) + (tw[2] + tw[3]))};
        if (k > 0) {
            // Candidates: what beats the wave's k-th so far, and is not below the k-th largest of the
            // lanes' maxima (at least k values of this tile are no smaller), whose upper 16 bits a
            // binary search over the lanes finds.
            uint32_t from = (uint32_t)(top.kth >> 32);
            if (!__any(!(m <= value_of(from)))) continue;
            const uint32_t p = reached_by(k, order_of(m));
            if (p > 0 && p - 1 > from) from = p - 1;
            const float f = value_of(from == 0x7fffffffu ? 0x7ffffffeu : from);      // no -0: it would equal +0
            uint32_t in = 0;
#pragma unroll
            for (int j = 0; j < kLpTile; j++) in |= !(v[j] <= f) ? 1u << j : 0u;
            while (__any(in != 0)) {               // mostly one or two a lane: read again, not kept by a register index
                unsigned long long key[4];
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    const int j = in ? __builtin_ctz(in) : 0, i = t0 + ((j / VEC) * 64 + lane) * VEC + j % VEC;
                    key[n] = in != 0 && i < v1 ? key_of((float)row[i], i) : 0;
                    in &= in - 1;
                }
#pragma unroll
                for (int n = 0; n < 4; n++) top_add(top, key[n] > top.kth, key[n]);
            }
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        stats b = {__shfl_xor(a.m, o), __shfl_xor(a.s, o), __shfl_xor(a.w, o)};
        join(a, b);
    }
    if (lane == 0) red[wave] = a;
    if (k > 0) {
        top_flush(top);
        lds_sync();
        top.wait[lane] = top.best;
    }
    __syncthreads();
    if (wave != 0) return;
    const size_t u = (size_t)r * C + c;
    if (lane == 0) {
        for (int w = 1; w < 4; w++) join(a, red[w]);
        part[4 * u] = a.m;
        part[4 * u + 1] = a.s;
        part[4 * u + 2] = a.w;
    }
    if (k > 0) {
        for (int w = 1; w < 4; w++) top.best = merge_down(top.best, lists[w][63 - lane]);
        if (lane < k) keys[u * k + lane] = top.best;
    }
}

// Row r's results from its C parts: 64 threads.  Bound: two dependent rounds of loads, then the alternatives (one
// row of 19 parts: 2.1 us without, 4.3 us with 20, 8 us with 64).
template <typename X>
__device__ __forceinline__ void lp_join(const X* __restrict__ x, long long xs, int V, int C, const int* __restrict__ tok,
                                        int nt, float* __restrict__ logp, float* __restrict__ entropy, int k,
                                        float* __restrict__ top_logp, int* __restrict__ top_id,
                                        const float* __restrict__ part, const unsigned long long* __restrict__ keys) {
    __shared__ unsigned long long list[kTop + 64];
    const int lane = threadIdx.x, r = blockIdx.x;
    const X* row = x + (long long)r * xs;
    stats a = {-3.402823466e38f, 0.0f, 0.0f};
    for (int c = lane; c < C; c += 64) {
        const float* p = part + 4 * ((size_t)r * C + c);
        join(a, stats{p[0], p[1], p[2]});
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        stats b = {__shfl_xor(a.m, o), __shfl_xor(a.s, o), __shfl_xor(a.w, o)};
        join(a, b);
    }
    // S == 0: every logit is -infinity, there is nothing to share out: log probabilities -infinity,
    // entropy 0.  S not a number: the row holds a NaN or +infinity.
    const float lz = logf(a.s);
    const bool none = a.s == 0.0f, odd = a.s != a.s;
    auto lp = [&](float v) { return none ? -INFINITY : (v - a.m) - lz; };
    if (entropy && lane == 0) entropy[r] = none ? 0.0f : lz - a.w / a.s * kLn2;
    for (int i = lane; i < nt; i += 64) {
        const int t = tok[(size_t)r * nt + i];
        logp[(size_t)r * nt + i] = t >= 0 && t < V ? lp((float)row[t]) : 0.0f;
    }
    if (k == 0) return;
    top_list top = {list, k, 0, 0, 0};
    const unsigned long long* kr = keys + (size_t)r * C * k;
    // Eight of the chunks' keys a lane at a time, every chunk's best before any's second; as above, what is
    // below the k-th largest of the lanes' best is none of the k best.
    for (int i0 = 0; i0 < C * k; i0 += 512) {
        unsigned long long key[8], most = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int i = i0 + 64 * j + lane;
            key[j] = i < C * k ? kr[i % C * k + i / C] : 0;
            most = key[j] > most ? key[j] : most;
        }
        const uint32_t p = reached_by(k, (uint32_t)(most >> 32));
#pragma unroll
        for (int j = 0; j < 8; j++) top_add(top, key[j] > top.kth && (uint32_t)(key[j] >> 32) >= p, key[j]);
    }
    top_flush(top);
    if (lane < k) {
        const unsigned long long key = top.best;
        top_id[(size_t)r * k + lane] = key && !odd ? (int)~(uint32_t)key : -1;
        top_logp[(size_t)r * k + lane] = odd ? a.s : key ? lp(value_of((uint32_t)(key >> 32))) : -INFINITY;
    }
}

// ---- attention over a shared prefix ----
}  // namespace

// What the launcher passes by value: sgpu_attn_prefix_args (include/switch_gpu.h) without its hints, and the
// plan.  The prefix is NKV * MTp units (KV head, row tile) of `stages` steps of `step` keys; its nbp blocks take
// `run` of all units' steps each (fewer than 2^30), so a unit is spread over some blocks, its splits (at most Sp), and a
// block may end one unit and begin the next.  A sequence's own keys: B * NKV by MTs row tiles and Ss splits.
struct attn_prefix {
    const void *q, *kp, *vp, *ks, *vs;
    float* out;
    const int *q_start, *kv_start, *kv_len;
    float *po, *pml;                  // partial outputs, and (max, sum, mark, -) of each: [split][row][head]
    long long q_row, q_head, out_row, out_head, kp_row, kp_head, ks_row, ks_head;
    int R, B, P, SR, NH, NKV;
    float scale;
    int Sp, stages, step, run, MTp, nbp, nbs, MTs, Ss, wide_p, wide_s;   // run: a block's steps; nbs: the own keys' blocks
    _Float16* cut;                    // attn_cut's pieces and scales
    int* scales;
};

namespace {

constexpr int kSpread = 10;           // binary orders within which the keys of a group share a scale
constexpr int kLeastV = -64, kMostV = 32;      // scales of V that the running sums bear beside each other (attn_unit)

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    auto step = [&](uint32_t o) { v = o > v ? o : v; };
    step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, SGPU_DPP_ROW_SHR(1), 0xf, 0xf, true));
    step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, SGPU_DPP_ROW_SHR(2), 0xf, 0xf, true));
    step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, SGPU_DPP_ROW_SHR(4), 0xf, 0xf, true));
    step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, SGPU_DPP_ROW_SHR(8), 0xf, 0xf, true));
    step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, SGPU_DPP_ROW_BCAST15, 0xa, 0xf, true));
    step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, SGPU_DPP_ROW_BCAST31, 0xc, 0xf, true));
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
template <typename KV> struct cache;
template <> struct cache<float> { static constexpr int PIECES = 2; };
template <> struct cache<_Float16> { static constexpr int PIECES = 1; };

struct attn_info { int kexp[4], vexp[4], oddk[4], oddv[4]; };     // of a tile's 16-key groups

// Rows (query row, head of the group) against keys k0 .. k1-1 of one KV head, on the fp16 matrix cores.
//
// fp32 operands are cut into two fp16 pieces with a power of two as scale (q: one a row; K and V: one
// for each 16 keys, 32 where cut ahead), of whose four products the three larger ones are summed in fp32: 22 bits of
// every operand (2^-36 of the largest that shares its scale, where that is more), what is left out is below 2^-22 of a
// product.  fp16 caches are one piece, exact.
// Softmax weights are cut the same way: P = 2^(x + e - M + OFF), x the score in powers of two, e the scale of
// the key's V, M the row's largest x + e so far or up to 2^LAG below it (so that O, which the matrix cores
// add to in place, is hardly ever scaled again).  A weight is off by 2^(-25-OFF) of the largest term's; the
// sum l of 2^(x - m) is taken from P before it is cut, as P 2^(M - m - OFF - e).  Both factors hold V's scale, so scales
// are kept to kLeastV .. kMostV: a key d binary orders below m then has P = 2^(8 + e - max e - d) or more, a normal number
// down to d = 38, and M - m stays within the scales and LAG of each other.  (Values of a group up to 2^-53 to 2^47.  fp16
// values have no scale, so OFF is as large as fp16's range allows: 2^-39 beside values of up to 2^16.)
// Keys of one group whose sizes lie more than 2^kSpread apart must not share a scale, a group of zero values
// has none, one of values past those sizes none that may be used, and a value that is not a number must not meet the zero
// weight of a row that does not see it: 32 keys with such a group are left out here, the record marked, and taken by
// attn_join on the vector ALUs in fp32 (odd_tiles).
//
// A block is four waves of 32 rows that share tiles of KT keys (WR = 4), or four waves of the same 32
// rows, each with its own 32 keys at a time, merged at the end (WR = 1).  Both products run transposed, so that
// a lane holds one row: S^T = K Q^T (accumulator r: key 8*(r/4) + 4*h + r%4 of 32, row l32), O^T =
// V^T P^T, whose B operand, P, lies where the first product left it: the order of the keys within a
// 16-key step is free, and V^T is stored for this one.
//
// Bound: many rows, the matrix cores and the vector ALUs together.  32 rows by 32 keys of 64 dims in pieces are 24
// products (386 ns of a SIMD) and some 115 vector instructions with 16 exponentials (370 ns), which run side by
// side in part: a SIMD with three waves takes 640 ns.  34080 rows and heads over 3001 keys (fp32, 64 dims): 91 us, 0.86
// PFLOP/s of piece products (large fp16 products of the library reach 1.1 here); without the exponentials and
// cuts 79, without the maxima 80, with tiles of zeros 75.  1536 rows and heads over 32768 fp16 keys (8 KV heads
// of 128 dims, 134 MB): 82 us.  Few rows, latency: a block takes 0.8 us to its first load, 1.4 to its rows, 2.3 for each step
// of 128 keys and 1.9 to merge and write (4 rows of 14 heads over 500 keys: 8.0 us).
template <int HD, typename KV, int WR> struct attn_unit {
    static constexpr int NP = cache<KV>::PIECES, DW = HD / 16, ND = HD / 32, NK = HD / 16;
    static constexpr float OFF = NP == 2 ? 8.0f : 14.0f, LAG = NP == 2 ? 7.0f : 1.0f;      // P up to 2^15
    static constexpr int KT = WR == 1 ? 32 : HD > 64 ? 32 : 64, NG = KT / 16;
    // LDS: K pieces [piece][key][HD], V pieces [piece][dim][KT], 16-byte chunks swizzled so that 16 lanes'
    // chunks of a column use all banks; WR = 1 keeps one region per wave, K first, then V.
    static constexpr int PART = NP * KT * HD;                      // halves of K or of V
    static constexpr int NCK = HD / 8, RPK = NCK < 16 ? 16 / NCK : 1, NCV = KT / 8, RPV = 16 / NCV;
    static constexpr int BYTES_TILES = WR == 1 ? 4 * PART * 2 : 2 * 2 * PART * 2;
    static constexpr int BYTES_MERGE = WR == 1 ? 4 * 32 * (HD + 1) * 4 + 4 * 2 * 32 * 4 : 0;
    static constexpr int BYTES = BYTES_TILES > BYTES_MERGE ? BYTES_TILES : BYTES_MERGE;

    typedef KV vec __attribute__((ext_vector_type(DW)));
    struct block { vec v[4]; };                                    // 4 keys by DW dims
    static constexpr int ROWS = WR == 1 ? 32 : 128;

    const attn_prefix& a;
    _Float16* tiles;
    attn_info* inf;                                                    // WR = 4: two, by buffer
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l32 = lane & 31, h = lane >> 5, dq = lane & 15, kq = lane >> 4;

    const KV *K, *V;                                               // key 0
    int row;                                                       // values from key to key
    int k0, k1, seen;                                              // seen: keys this lane's row sees (of all)
    bool own;                                                      // a sequence's own keys, not all of them seen by all rows
    int qx;                                                        // the row's scale: q is pieces * 2^qx
    f16x8 q[2][NK];
    f32x16 o[ND];
    float m, M, l, A;                                              // A = 2^(M - m - OFF)

    __device__ __forceinline__ attn_unit(const attn_prefix& a_, _Float16* t, attn_info* i) : a(a_), tiles(t), inf(i) {}

    // ---- staging ----
    __device__ __forceinline__ void load(block& b, const KV* X, int key) const {       // 16 keys from `key`
        typedef KV mem __attribute__((ext_vector_type(DW), aligned(DW * sizeof(KV) < 16 ? DW * sizeof(KV) : 16)));
        const KV* p = X + (long long)key * row;
        const int last = k1 - 1 - key;                             // rows past the end repeat the last one
        const int at = 4 * kq * row + dq * DW;
        if (last < 15) {
#pragma unroll
            for (int i = 0; i < 4; i++) b.v[i] = *reinterpret_cast<const mem*>(p + (min(4 * kq + i, last) * row + dq * DW));
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) b.v[i] = *reinterpret_cast<const mem*>(p + (at + i * row));
        }
    }
    // Keys from the end on become zeros.
    __device__ __forceinline__ void trim(block& b, int key) const {
        if (k1 - key >= 16) return;
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (4 * kq + i >= k1 - key) b.v[i] = vec(0);
    }
    // The scale of a group of B * 16 keys from `key` on; odd: not one scale for it all.  Parts of a key that lie
    // near the largest spare the search for each key's own.
    template <bool IS_V, int B> __device__ __forceinline__ int survey(const block (&b)[B], int key, bool& odd) const {
        odd = false;
        if constexpr (NP == 1) {                                   // fp16 is used as it is
            if (IS_V && own) {
                bool bad = false;
#pragma unroll
                for (int n = 0; n < 4 * B; n++)
#pragma unroll
                    for (int e = 0; e < DW; e++) bad |= !__builtin_isfinite((float)b[n / 4].v[n % 4][e]);
                odd = __any(bad);
            }
            return 0;
        } else {
            float mx[4 * B], most = 0.0f;
            bool nan = false;
#pragma unroll
            for (int n = 0; n < 4 * B; n++) {
                mx[n] = fabsf(b[n / 4].v[n % 4][0]);
#pragma unroll
                for (int e = 1; e < DW; e++) mx[n] = fmaxf(mx[n], fabsf(b[n / 4].v[n % 4][e]));
                most = fmaxf(most, mx[n]);
            }
            const uint32_t top = wave_max_u32(__float_as_uint(most));
            if (IS_V && own) {                                     // fmaxf passes over NaN
#pragma unroll
                for (int n = 0; n < 4 * B; n++)
#pragma unroll
                    for (int e = 0; e < DW; e += 2) nan |= __builtin_isunordered(b[n / 4].v[n % 4][e], b[n / 4].v[n % 4][e + 1]);
                nan = __any(nan);
            }
            odd = nan || top >= 0x7f800000u || (IS_V && top == 0 && key < k1);
            uint32_t least = 0xffffffffu;
#pragma unroll
            for (int n = 0; n < 4 * B; n++) least = min(least, __float_as_uint(mx[n]) - 1u);   // zeros pass as the largest number
            if (!odd && __any(least < top && least + (kSpread << 23) < top)) {
                bool far = false;
#pragma unroll
                for (int n = 0; n < 4 * B; n++) {
                    uint32_t x = __float_as_uint(mx[n]);
#pragma unroll
                    for (int o = 1; o < 16; o *= 2) x = max(x, (uint32_t)__shfl_xor((int)x, o));
                    far |= x - 1u < top && x + (kSpread << 23) < top;
                }
                odd = __any(far);
            }
            const int ex = scale_of(top);
            if (IS_V) odd |= ex < kLeastV || ex > kMostV;
            return ex;
        }
    }
    __device__ __forceinline__ void put_k(_Float16* Kt, const block& b, int grp, int ex) const {
        const float up = pow2(-ex);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int key = 16 * grp + 4 * kq + i, d = dq * DW;
            _Float16* p = Kt + key * HD + 8 * ((d / 8) ^ ((key / RPK) % NCK)) + d % 8;
#pragma unroll
            for (int e = 0; e < DW; e += 2) {
                if constexpr (NP == 2) {
                    f16x2 hi, lo;
                    split2((float)b.v[i][e] * up, (float)b.v[i][e + 1] * up, hi, lo);
                    *reinterpret_cast<f16x2*>(p + e) = hi;
                    *reinterpret_cast<f16x2*>(p + KT * HD + e) = lo;
                } else {
                    *reinterpret_cast<f16x2*>(p + e) = f16x2{(_Float16)b.v[i][e], (_Float16)b.v[i][e + 1]};
                }
            }
        }
    }
    __device__ __forceinline__ void put_v(_Float16* Vt, const block& b, int grp, int ex) const {
        const float up = pow2(-ex);
#pragma unroll
        for (int e = 0; e < DW; e++) {
            const int d = dq * DW + e, c = 2 * grp + (kq & 1);
            _Float16* p = Vt + d * KT + 8 * (c ^ (((d / RPV) ^ (d / 16)) % NCV)) + 4 * (kq >> 1);
            if constexpr (NP == 2) {
                f16x2 hi[2], lo[2];
#pragma unroll
                for (int i = 0; i < 2; i++) split2((float)b.v[2 * i][e] * up, (float)b.v[2 * i + 1][e] * up, hi[i], lo[i]);
                *reinterpret_cast<f16x4*>(p) = f16x4{hi[0][0], hi[0][1], hi[1][0], hi[1][1]};
                *reinterpret_cast<f16x4*>(p + KT * HD) = f16x4{lo[0][0], lo[0][1], lo[1][0], lo[1][1]};
            } else {
                *reinterpret_cast<f16x4*>(p) =
                    f16x4{(_Float16)b.v[0][e], (_Float16)b.v[1][e], (_Float16)b.v[2][e], (_Float16)b.v[3][e]};
            }
        }
    }

    // ---- 32 keys (subtile u of the tile) ----
    // T keys a tile: KT, or 32 of the fp16 tiles
    template <int T> __device__ __forceinline__ f32x16 scores(const _Float16* Kt, int u) const {
        constexpr int C = HD > 64 && NP == 2 ? NK / 2 : NK;        // columns of K fragments held at a time
        const int key = 32 * u + l32;
        f32x16 s;
#pragma unroll
        for (int r = 0; r < 16; r++) s[r] = 0.0f;
#pragma unroll
        for (int k0 = 0; k0 < NK; k0 += C) {
            f16x8 f[C][NP];
#pragma unroll
            for (int k = 0; k < C; k++)
#pragma unroll
                for (int p = 0; p < NP; p++)
                    f[k][p] = *reinterpret_cast<const f16x8*>(Kt + p * T * HD + key * HD + 8 * ((2 * (k0 + k) + h) ^ ((key / RPK) % NCK)));
            __builtin_amdgcn_sched_barrier(0);                     // all loads out before the first product waits
#pragma unroll
            for (int k = 0; k < C; k++) {
                if constexpr (NP == 2) s = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[k][1], q[0][k0 + k], s, 0, 0, 0);
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[k][0], q[1][k0 + k], s, 0, 0, 0);
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[k][0], q[0][k0 + k], s, 0, 0, 0);
            }
        }
        return s;
    }
    __device__ __forceinline__ f16x8 v_at(const _Float16* Vt, int p, int j, int grp) const {
        const int d = 32 * j + l32;
        return *reinterpret_cast<const f16x8*>(Vt + p * KT * HD + d * KT + 8 * ((2 * grp + h) ^ (((d / RPV) ^ (d / 16)) % NCV)));
    }
    // Scores of 32 keys from `key` on: those that the row does not see masked, and the running statistics.  E: scales
    // of 16 keys each, or one; f: the scores' factors by scale.
    template <int E> __device__ __forceinline__ void factors(const int (&kexp)[E], float (&f)[E]) const {
#pragma unroll
        for (int g = 0; g < E; g++)                                // neither 0 nor infinite: it multiplies masked scores
            f[g] = fminf(fmaxf(__builtin_amdgcn_ldexpf(a.scale * kLog2e, qx + kexp[g]), 1.17549435e-38f), 3.402823466e38f);
    }
    template <int E> __device__ __forceinline__ void tops(const f32x16& s, float (&top)[E]) const {
        constexpr int N = 16 / E;
#pragma unroll
        for (int g = 0; g < E; g++) {
            top[g] = s[N * g];
#pragma unroll
            for (int r = 1; r < N; r++) top[g] = fmaxf(top[g], s[N * g + r]);
        }
    }
    template <int E> __device__ __forceinline__ void maxima(f32x16& s, int key, const int (&vexp)[E], const float (&f)[E]) {
        float top[E];
        tops(s, top);
        maxima(s, top, key, vexp, f);
    }
    template <int E>
    __device__ __forceinline__ void maxima(f32x16& s, float (&top)[E], int key, const int (&vexp)[E], const float (&f)[E]) {
        const int rest = seen - key;                               // how many of the keys the row sees
        if (__any(rest < 32)) {
#pragma unroll
            for (int r = 0; r < 16; r++)
                if (8 * (r / 4) + 4 * h + r % 4 >= rest) s[r] = -INFINITY;
            tops(s, top);
        }
        float tx, tz;
#pragma unroll
        for (int g = 0; g < E; g++) {
            const float t = top[g] * f[g];
            const float z = t + (float)vexp[g];
            tx = g ? fmaxf(tx, t) : t;
            tz = g ? fmaxf(tz, z) : z;
        }
        tx = half_max(tx);
        tz = E == 1 ? tx + (float)vexp[0] : half_max(tz);
        if (__any(tx > m + LAG || tz > M + LAG)) {                 // mostly at the first keys only
            const float mn = fmaxf(m, tx), Mn = fmaxf(M, tz);
            const float al = __builtin_amdgcn_exp2f(M - Mn);
            l *= __builtin_amdgcn_exp2f(m - mn);
#pragma unroll
            for (int j = 0; j < ND; j++)
#pragma unroll
                for (int r = 0; r < 16; r++) o[j][r] *= al;
            m = mn;
            M = Mn;
            A = __builtin_amdgcn_exp2f(M - m - OFF);
        }
    }
    // ... to weights, as pieces by 16-key step
    template <int E>
    __device__ __forceinline__ void weights(const f32x16& s, const int (&vexp)[E], const float (&f)[E], f16x8 (&ph)[2], f16x8 (&pl)[2]) {
        constexpr int N = 16 / E;
#pragma unroll
        for (int g = 0; g < E; g++) {
            const float b = ((float)vexp[g] + OFF) - M;
            float sum = 0.0f;
#pragma unroll
            for (int r = N * g; r < N * (g + 1); r += 2) {
                const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], f[g], b));
                const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r + 1], f[g], b));
                sum += p0;
                sum += p1;
                f16x2 hi, lo;
                split2(p0, p1, hi, lo);
                ph[r / 8][r % 8] = hi[0];
                ph[r / 8][r % 8 + 1] = hi[1];
                pl[r / 8][r % 8] = lo[0];
                pl[r / 8][r % 8 + 1] = lo[1];
            }
            l = __builtin_fmaf(sum, __builtin_amdgcn_ldexpf(A, -vexp[g]), l);
        }
    }
    // O += V^T P^T of 32 keys; at(piece, dims / 32, 16-key step): V^T
    template <typename F> __device__ __forceinline__ void values(F at, const f16x8 (&ph)[2], const f16x8 (&pl)[2]) {
#pragma unroll
        for (int g = 0; g < 2; g++)
#pragma unroll
            for (int j = 0; j < ND; j++) {
                const f16x8 hi = at(0, j, g);
                if constexpr (NP == 2) o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(at(1, j, g), ph[g], o[j], 0, 0, 0);
                o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(hi, pl[g], o[j], 0, 0, 0);
                o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(hi, ph[g], o[j], 0, 0, 0);
            }
    }

    // ---- the unit ----
    const float* q_at;                                             // this lane's row
    __device__ __forceinline__ void load_q() {                     // its scale joins the softmax's
        const float* const x = q_at;
        float v[NK][8];
        uint32_t mx = 0;
#pragma unroll
        for (int k = 0; k < NK; k++)
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const sgpu_f32x4 w = *reinterpret_cast<const sgpu_f32x4*>(x + 16 * k + 8 * h + e);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    v[k][e + i] = w[i];
                    const uint32_t b = __float_as_uint(w[i]) & 0x7fffffffu;
                    mx = max(mx, b < 0x7f800000u ? b : 0u);
                }
            }
        mx = max(mx, (uint32_t)__shfl_xor((int)mx, 32));
        qx = scale_of(mx);
        const float up = pow2(-qx);
#pragma unroll
        for (int k = 0; k < NK; k++)
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                f16x2 hi, lo;
                split2(v[k][e] * up, v[k][e + 1] * up, hi, lo);
                q[0][k][e] = hi[0];
                q[0][k][e + 1] = hi[1];
                q[1][k][e] = lo[0];
                q[1][k][e + 1] = lo[1];
            }
        clear();
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int j = 0; j < ND; j++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[j][r] = 0.0f;
        m = M = -3e38f;                                            // finite: what it is subtracted from may be -infinity
        l = 0.0f;
        A = pow2((int)-OFF);
    }

    // WR = 4: a wave stages K and V of group `wave` (KT 64), or K or V of one of two groups (KT 32).
    struct staged { block k[1], v[1]; };
    __device__ __forceinline__ void fetch(staged& st, int key) const {
        if constexpr (NG == 4) {
            load(st.k[0], K, key + 16 * wave);
            load(st.v[0], V, key + 16 * wave);
        } else {
            load(st.k[0], wave < 2 ? K : V, key + 16 * (wave & 1));
        }
    }
    __device__ __forceinline__ void stage(staged& st, int key, _Float16* Kt, _Float16* Vt, attn_info& f) const {
        const int g = NG == 4 ? wave : wave & 1;
        bool oddk = false, oddv = false;
        trim(st.k[0], key + 16 * g);
        if constexpr (NG == 4) {
            trim(st.v[0], key + 16 * g);
            const int ke = survey<false>(st.k, key + 16 * g, oddk), ve = survey<true>(st.v, key + 16 * g, oddv);
            put_k(Kt, st.k[0], g, ke);
            put_v(Vt, st.v[0], g, ve);
            if (lane == 0) {
                f.kexp[g] = ke;
                f.vexp[g] = ve;
                f.oddk[g] = oddk;
                f.oddv[g] = oddv;
            }
        } else if (wave < 2) {
            const int ke = survey<false>(st.k, key + 16 * g, oddk);
            put_k(Kt, st.k[0], g, ke);
            if (lane == 0) {
                f.kexp[g] = ke;
                f.oddk[g] = oddk;
            }
        } else {
            const int ve = survey<true>(st.k, key + 16 * g, oddv);
            put_v(Vt, st.k[0], g, ve);
            if (lane == 0) {
                f.vexp[g] = ve;
                f.oddv[g] = oddv;
            }
        }
    }
    __device__ __forceinline__ bool run_shared() {                 // true: something was odd
        const int nt = (k1 - k0 + KT - 1) / KT;
        bool any = false;
        staged st;
        fetch(st, k0);
        load_q();                                                  // under the first keys' way
        stage(st, k0, tiles, tiles + PART, inf[0]);
        if (nt > 1) fetch(st, k0 + KT);
        for (int t = 0; t < nt; t++) {
            const int key = k0 + t * KT;
            const _Float16* const Kt = tiles + (t & 1) * 2 * PART;
            const attn_info& f = inf[t & 1];
            __syncthreads();                                       // the tile is in LDS, the other buffer free
#pragma unroll
            for (int u = 0; u < KT / 32; u++) {
                int kexp[2], vexp[2], odd = 0;
#pragma unroll
                for (int g = 0; g < 2; g++) {
                    kexp[g] = __builtin_amdgcn_readfirstlane(f.kexp[2 * u + g]);
                    vexp[g] = __builtin_amdgcn_readfirstlane(f.vexp[2 * u + g]);
                    odd |= f.oddk[2 * u + g] | f.oddv[2 * u + g];
                }
                if (__builtin_amdgcn_readfirstlane(odd)) {
                    any = true;
                    continue;
                }
                f32x16 s = scores<KT>(Kt, u);
                f16x8 ph[2], pl[2];
                float f[2];
                factors(kexp, f);
                maxima(s, key + 32 * u, vexp, f);
                weights(s, vexp, f, ph, pl);
                values([&](int p, int j, int g) { return v_at(Kt + PART, p, j, 2 * u + g); }, ph, pl);
            }
            if (t + 1 < nt) {
                _Float16* const Kn = tiles + ((t + 1) & 1) * 2 * PART;
                stage(st, key + KT, Kn, Kn + PART, inf[(t + 1) & 1]);
                if (t + 2 < nt) fetch(st, key + 2 * KT);
            }
        }
        return any;
    }
    // ---- tiles that come as fp16 rows: an fp16 cache, or the pieces that attn_cut made of an fp32 one ----
    // Row-major tiles of 32 keys go straight into LDS (16 bytes a lane, no registers) through a ring of RING
    // tiles for K and one for V.  K chunks are swizzled as above, V rows by 64 bytes, so that the transposing
    // reads (4 keys by 16 dims for 16 lanes) of 8 keys use all banks.  The products of the next
    // tile's scores run under this tile's exponentials: in step t the block uses V of tile t and K of tile t + 1.
    static constexpr int DPART = NP * 32 * HD, RPI = 512 / HD, PW = NP * HD / 32;      // loads of a wave and tile
    static constexpr int RING = HD * NP >= 256 ? 2 : HD * NP == 128 && NP == 2 ? 3 : 4, BYTES_DIRECT = 2 * RING * DPART * 2;
    static __device__ __forceinline__ int v_chunk(int c, int key) {            // 16-byte chunk c of a row of V
        return HD == 32 ? c : HD == 64 ? c ^ (4 * ((key >> 1) & 1)) : c ^ (4 * (key & 3));
    }
    struct source {
        const _Float16 *k, *v;                                     // key 0 of piece 0
        long long piece;                                           // values from piece to piece
        int row;                                                   // values from key to key
        const int* scales;                                         // (K's, V's exponent, odd, -) of each 32 keys; NP 2
    };
    // A wave's loads of a tile: RPI rows of a piece each, (K's pieces, V's pieces) by row blocks dealt to the four
    // waves in turn.  V comes a tile behind K.  Rows past the end read as zeros, and so do whole tiles past
    // it: the number of loads is always PW.
    static constexpr int RB = HD / 16;                             // row blocks of a piece
    struct loader {
        uint64_t from[PW];
        int offset[PW], at[PW], left[2], row;                      // left: K's, V's keys from the next tile on
    };
    __device__ __forceinline__ void start(loader& ld, const source& x) const {
        const int r = lane / (HD / 8), c = lane % (HD / 8);
        const uint32_t base = (uint32_t)(uintptr_t)(lds_void*)tiles;
#pragma unroll
        for (int i = 0; i < PW; i++) {
            const int n = 4 * i + wave, part = n / RB, block = n % RB, piece = part % NP, key = block * RPI + r;
            const bool is_v = part >= NP;
            ld.from[i] = (uint64_t)((is_v ? x.v : x.k) + piece * x.piece + (long long)(k0 - (is_v ? 32 : 0)) * x.row);
            ld.at[i] = base + 2 * ((is_v ? RING * DPART : 0) + piece * (32 * HD) + block * (RPI * HD));
            ld.offset[i] = (key * x.row + 8 * (is_v ? v_chunk(c, key) : c ^ ((key / RPK) % NCK))) * 2;
        }
        ld.left[0] = k1 - k0;
        ld.left[1] = k1 - k0 + 32;
        ld.row = x.row;
    }
    // The next tile of K into place `place` of its ring, the next of V into the place before it (FIRST: none yet).
    template <bool FIRST = false> __device__ __forceinline__ void fetch_direct(loader& ld, int place) const {
#pragma unroll
        for (int i = 0; i < PW; i++) {
            const bool is_v = (4 * i + wave) / RB >= NP;
            const int left = ld.left[is_v], rows = min(left, 32), to = is_v ? (place > 0 ? place - 1 : RING - 1) : place;
            const int bytes = rows > 0 && !(FIRST && is_v) ? ((rows - 1) * ld.row + HD) * 2 : 0;
            // As asm, which the compiler does not wait for at the next LDS read: run_direct waits before its
            // barriers.  (No output registers; m0 holds the LDS address, and nothing else here uses it.)
            const i32x4 rsrc = {(int)ld.from[i], (int)(ld.from[i] >> 32) & 0xffff, bytes, 0x00020000};
            __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                             :
                             : "s"(ld.at[i] + to * DPART * 2), "v"(ld.offset[i]), "s"(rsrc)
                             : "memory");
            ld.from[i] += (uint64_t)(64 * ld.row);
        }
        ld.left[0] -= 32;
        ld.left[1] -= 32;
    }
    template <int LEFT> static __device__ __forceinline__ void landed() {      // all but the last LEFT loads
        __asm__ volatile("s_waitcnt vmcnt(%0)" : : "i"(LEFT) : "memory");
        __syncthreads();
    }
    // V^T of 16 keys and 32 dims: lane (dim l32, h) gets keys 4 h .. and 8 + 4 h .. of the 16.
    __device__ __forceinline__ f16x8 v_direct(const _Float16* Vt, int p, int j, int g) const {
        const int i = lane & 15, d = 32 * j + 16 * ((lane >> 4) & 1) + 4 * (i & 3);
        f16x8 r;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int key = 16 * g + 8 * e + 4 * h + (i >> 2);
            const _Float16* at = Vt + p * 32 * HD + key * HD + 8 * v_chunk(d / 8, key) + d % 8;
            const s16x4 w = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at);
            const f16x4 x = __builtin_bit_cast(f16x4, w);
#pragma unroll
            for (int k = 0; k < 4; k++) r[4 * e + k] = x[k];
        }
        return r;
    }
    // A step: the weights from `s`, the scores of the next tile, and O += weights times V.  The order is written
    // out, a barrier to the compiler's scheduler after each piece: vector instructions between the products, and
    // LDS reads two fragments ahead of their use.  top: of the next scores.
    __device__ __forceinline__ f32x16 step(const _Float16* Kt, const _Float16* Vt, const f32x16& s, int vexp, float f, float& top) {
        constexpr int L = NK + 2 * ND, PER = 8 / NK > 0 ? 8 / NK : 1;      // fragments; pairs of weights a K fragment
        const float b = ((float)vexp + OFF) - M;
        float sum = 0.0f, t = 0.0f;
        f16x8 fr[L][NP], ph[2], pl[2];
        f32x16 n;
#pragma unroll
        for (int r = 0; r < 16; r++) n[r] = 0.0f;
        auto read = [&](int i) __attribute__((always_inline)) {
#pragma unroll
            for (int p = 0; p < NP; p++)
                if (i < NK) fr[i][p] = *reinterpret_cast<const f16x8*>(Kt + p * 32 * HD + l32 * HD + 8 * ((2 * i + h) ^ ((l32 / RPK) % NCK)));
                else if (i < L) fr[i][p] = v_direct(Vt, p, (i - NK) % ND, (i - NK) / ND);
        };
        read(0);
        read(1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < NK; i++) {
            float w[PER][2];
            f16x2 hi[PER], lo[PER];
            read(i + 2);
            if constexpr (NP == 2) {
                n = __builtin_amdgcn_mfma_f32_32x32x16_f16(fr[i][1], q[0][i], n, 0, 0, 0);
            } else {
                n = __builtin_amdgcn_mfma_f32_32x32x16_f16(fr[i][0], q[1][i], n, 0, 0, 0);
            }
#pragma unroll
            for (int x = 0; x < PER; x++)
#pragma unroll
                for (int e = 0; e < 2; e++) w[x][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * (PER * i + x) + e], f, b));
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (NP == 2) {
                n = __builtin_amdgcn_mfma_f32_32x32x16_f16(fr[i][0], q[1][i], n, 0, 0, 0);
#pragma unroll
                for (int x = 0; x < PER; x++) sum += w[x][0];
#pragma unroll
                for (int x = 0; x < PER; x++) sum += w[x][1];
                __builtin_amdgcn_sched_barrier(0);
            }
            n = __builtin_amdgcn_mfma_f32_32x32x16_f16(fr[i][0], q[0][i], n, 0, 0, 0);
#pragma unroll
            for (int x = 0; x < PER; x++) {
                const int r = 2 * (PER * i + x);
                split2(w[x][0], w[x][1], hi[x], lo[x]);
                if constexpr (NP == 1) sum = sum + w[x][0] + w[x][1];
                ph[r / 8][r % 8] = hi[x][0];
                ph[r / 8][r % 8 + 1] = hi[x][1];
                pl[r / 8][r % 8] = lo[x][0];
                pl[r / 8][r % 8 + 1] = lo[x][1];
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        l = __builtin_fmaf(sum, __builtin_amdgcn_ldexpf(A, -vexp), l);
#pragma unroll
        for (int i = NK; i < L; i++) {
            const int j = (i - NK) % ND, g = (i - NK) / ND;
            read(i + 2);
            if constexpr (NP == 2) o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fr[i][1], ph[g], o[j], 0, 0, 0);
            o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fr[i][0], pl[g], o[j], 0, 0, 0);
            o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fr[i][0], ph[g], o[j], 0, 0, 0);
            constexpr int Z = 16 / (2 * ND);
#pragma unroll
            for (int r = Z * (i - NK); r < Z * (i - NK + 1); r++) t = r == 0 ? n[0] : fmaxf(t, n[r]);
            __builtin_amdgcn_sched_barrier(0);
        }
        top = t;
        return n;
    }
    __device__ __forceinline__ bool run_direct(const source& x) {
        const int nt = (k1 - k0 + 31) / 32;
        const bool idle = v0 + 32 * wave >= nv;                    // no rows of its own: it brings keys only
        typedef const int __attribute__((address_space(4)))* const_int;
        const_int sc = (const_int)(uintptr_t)x.scales + k0 / 32 * 4;
        bool any = false;
        loader ld;
        start(ld, x);
        fetch_direct<true>(ld, 0);
#pragma unroll 1
        for (int t = 1; t < RING; t++) fetch_direct(ld, t);
        load_q();                                                  // (waits for its own loads, and so for those before)
        landed<(RING - 1) * PW>();                                 // tile 0 of K
        f32x16 s = scores<32>(tiles, 0);
        int kexp[1] = {0}, vexp[1] = {0}, last = 0;
        float f[1], top[1];
        factors(kexp, f);
        tops(s, top);
        // (not unrolled over the ring's places: a block often runs few steps, and code costs its first run)
        int place = 0;
#pragma unroll 1
        for (int t = 0; t < nt; t++) {
            landed<(RING - 2) * PW>();                             // tile t + 1 of K, tile t of V; step t - 1 is over
            fetch_direct(ld, place);
            const _Float16* const Vt = tiles + (RING + place) * DPART;
            place = place + 1 < RING ? place + 1 : 0;
            const _Float16* const Kt = tiles + place * DPART;
            if (idle) continue;
            if constexpr (NP == 2) {
                kexp[0] = sc[0];
                vexp[0] = sc[1];
                const int odd = sc[2];
                sc += 4;
                if (odd) {
                    any = true;
                    s = scores<32>(Kt, 0);
                    tops(s, top);
                    continue;
                }
                if (kexp[0] != last) {
                    last = kexp[0];
                    factors(kexp, f);
                }
            }
            maxima(s, top, k0 + 32 * t, vexp, f);
            s = step(Kt, Vt, s, vexp[0], f[0], top[0]);            // (after the last tile: of what is there, not used)
        }
        landed<0>();
        return any;
    }

    __device__ __forceinline__ bool run_alone() {
        constexpr bool AHEAD = HD <= 64;                           // the next keys while these are used: registers allowing
        bool any = false;
        block kb[2], vb[2];
        auto one = [](const block& b) __attribute__((always_inline)) -> const block(&)[1] { return reinterpret_cast<const block(&)[1]>(b); };
        auto fetch = [&](block (&b)[2], const KV* X, int key) __attribute__((always_inline)) {
#pragma unroll
            for (int g = 0; g < 2; g++) load(b[g], X, key + 16 * g);
        };
        int key = k0 + 32 * wave;
        if (key < k1) fetch(kb, K, key);
        load_q();
        for (; key < k1; key += 128) {
            int kexp[2], vexp[2];
            bool odd = false, is;
            if (AHEAD) fetch(vb, V, key);
#pragma unroll
            for (int g = 0; g < 2; g++) {
                trim(kb[g], key + 16 * g);
                kexp[g] = survey<false>(one(kb[g]), key + 16 * g, is);
                odd |= is;
            }
            lds_sync();
#pragma unroll
            for (int g = 0; g < 2; g++) put_k(tiles, kb[g], g, kexp[g]);
            if (AHEAD && key + 128 < k1) fetch(kb, K, key + 128);
            lds_sync();
            f32x16 s = scores<KT>(tiles, 0);
            if (!AHEAD) {
                __builtin_amdgcn_sched_barrier(0);                 // V's registers are K's
                fetch(vb, V, key);
            }
#pragma unroll
            for (int g = 0; g < 2; g++) {
                trim(vb[g], key + 16 * g);
                vexp[g] = survey<true>(one(vb[g]), key + 16 * g, is);
                odd |= is;
            }
            if (odd) {
                any = true;
                if (!AHEAD && key + 128 < k1) fetch(kb, K, key + 128);
                continue;
            }
            lds_sync();
#pragma unroll
            for (int g = 0; g < 2; g++) put_v(tiles, vb[g], g, vexp[g]);
            f16x8 ph[2], pl[2];
            if (!AHEAD) __builtin_amdgcn_sched_barrier(0);
            float f[2];
            factors(kexp, f);
            maxima(s, key, vexp, f);
            weights(s, vexp, f, ph, pl);
            lds_sync();
            values([&](int p, int j, int g) { return v_at(tiles, p, j, g); }, ph, pl);
            if (!AHEAD && key + 128 < k1) {
                __builtin_amdgcn_sched_barrier(0);
                fetch(kb, K, key + 128);
            }
        }
        return any;
    }

    // The block's rows: v0 .. of nv (row rbase + v / G, head g * G + v % G).  Own keys: row i of the unit's rows sees
    // len - nq + i + 1 keys of len.
    int g, rbase, nv, v0;
    __device__ __forceinline__ void begin(int g_, int rbase_, int nv_, int v0_, int len, int nq) {
        g = g_;
        rbase = rbase_;
        nv = nv_;
        v0 = v0_;
        const int G = a.NH / a.NKV, v = v0 + (WR == 1 ? 0 : 32 * wave) + l32, i = min(v, nv - 1) / G;
        seen = v >= nv ? 0 : own ? min(max(len - nq + i + 1, 0), len) : k1;
        q_at = (const float*)a.q + (rbase + i) * a.q_row + (g * G + min(v, nv - 1) - i * G) * a.q_head;
    }
    __device__ __forceinline__ bool run_staged() {
        if constexpr (WR == 1) return run_alone();
        else return run_shared();
    }
    // To the records of split sp, O and l relative to 2^m; mark: 1 or 3 where keys were left out (3: by scales of 32 keys), 2 (fp16
    // tiles of own keys) where the row's sums are not numbers: a value that it does not see may have done that.
    __device__ __forceinline__ void finish(int sp, int odd) {
        const int G = a.NH / a.NKV;
        l = half_sum(l);
        const float back = __builtin_amdgcn_exp2f(M - m - OFF);
#pragma unroll
        for (int j = 0; j < ND; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) o[j][e] *= back;
        if constexpr (WR == 1) {                                   // merge the waves: 8 threads a row, HD / 8 dims each
            float* part = reinterpret_cast<float*>(tiles - wave * PART);
            float* ml = part + 4 * 32 * (HD + 1);
            __syncthreads();
#pragma unroll
            for (int j = 0; j < ND; j++)
#pragma unroll
                for (int e = 0; e < 16; e++) part[(wave * 32 + l32) * (HD + 1) + 32 * j + 8 * (e / 4) + 4 * h + e % 4] = o[j][e];
            if (h == 0) {
                ml[wave * 64 + l32] = m;
                ml[wave * 64 + 32 + l32] = l;
            }
            const bool any_odd = __syncthreads_or(odd);
            const int w = threadIdx.x / 8, d0 = (threadIdx.x % 8) * (HD / 8), vw = v0 + w;
            if (vw < nv) {
                float top = -INFINITY, L = 0.0f, x[HD / 8];
                for (int k = 0; k < 4; k++) top = fmaxf(top, ml[k * 64 + w]);
#pragma unroll
                for (int e = 0; e < HD / 8; e++) x[e] = 0.0f;
                for (int k = 0; k < 4; k++) {
                    const float wt = __builtin_amdgcn_exp2f(ml[k * 64 + w] - top), lw = ml[k * 64 + 32 + w];
                    if (lw == 0.0f) continue;                      // this wave saw nothing of the row
                    L = __builtin_fmaf(lw, wt, L);
#pragma unroll
                    for (int e = 0; e < HD / 8; e++) x[e] = __builtin_fmaf(part[(k * 32 + w) * (HD + 1) + d0 + e], wt, x[e]);
                }
                const int iw = vw / G, hw = g * G + vw - iw * G, rw = rbase + iw;
                const size_t rec = ((size_t)sp * a.R + rw) * a.NH + hw;
                if (threadIdx.x % 8 == 0)
                    *reinterpret_cast<sgpu_f32x4*>(a.pml + 4 * rec) = sgpu_f32x4{top, L, any_odd ? 1.0f : 0.0f, 0.0f};
#pragma unroll
                for (int e = 0; e < HD / 8; e += 4)
                    *reinterpret_cast<sgpu_f32x4*>(a.po + rec * HD + d0 + e) = sgpu_f32x4{x[e], x[e + 1], x[e + 2], x[e + 3]};
            }
        } else {
            const int v = v0 + 32 * wave + l32;
            float mark = (float)odd;
            if (NP == 1 && own) {
                float sum = 0.0f;
#pragma unroll
                for (int j = 0; j < ND; j++)
#pragma unroll
                    for (int e = 0; e < 16; e++) sum += o[j][e] * 0.0f;
                if (half_sum(sum) != 0.0f) mark = 2.0f;
            }
            if (v >= nv) return;
            const int i = v / G, hd = g * G + v - i * G, r = rbase + i;
            const size_t rec = ((size_t)sp * a.R + r) * a.NH + hd;
            if (h == 0) *reinterpret_cast<sgpu_f32x4*>(a.pml + 4 * rec) = sgpu_f32x4{m, l, mark, 0.0f};
#pragma unroll
            for (int j = 0; j < ND; j++)
#pragma unroll
                for (int e = 0; e < 16; e += 4)
                    *reinterpret_cast<sgpu_f32x4*>(a.po + rec * HD + 32 * j + 2 * e + 4 * h) =
                        sgpu_f32x4{o[j][e], o[j][e + 1], o[j][e + 2], o[j][e + 3]};
        }
    }
};

// One of two kernel arguments, as values: choosing between their addresses puts both into scratch memory.
template <typename T> __device__ __forceinline__ T pick(bool first, T x, T y) {
    __asm__("" : "+s"(x));
    __asm__("" : "+s"(y));
    return first ? x : y;
}

// Sequence b's rows and own keys, cut to the buffers, and the keys of split ss for a row tile from v0 on
// (no row of the tile sees past its last one's).
struct seq_keys {
    int q0, nq, first, len;
    __device__ __forceinline__ void read(const attn_prefix& a, int b) {
        q0 = min(max(a.q_start[b], 0), a.R);
        nq = min(max(a.q_start[b + 1], q0), a.R) - q0;
        first = min(max(a.kv_start[b], 0), a.SR);
        len = min(max(a.kv_len[b], 0), a.SR - first);
    }
    __device__ __forceinline__ void range(const attn_prefix& a, int ss, int v0, int G, int& k0, int& k1) const {
        const int rows = a.wide_s ? 128 : 32, step = a.wide_s ? 64 : 128;
        const int chunk = ((len + a.Ss - 1) / a.Ss + step - 1) / step * step;
        const long long at = (long long)ss * chunk;
        k0 = at < len ? (int)at : len;
        k1 = min(max(len - nq + min(nq, (v0 + rows - 1) / G + 1), 0), min(len - k0, chunk) + k0);
        k1 = max(k1, k0);
    }
};

// How blocks take their keys: 32 rows a block (FEW), 128 rows and the keys as they come (ROWS), 128 rows and fp16
// tiles (DIRECT).
enum { FEW, ROWS, DIRECT };
template <int HD, typename KV, int HOW> struct attn_how {
    typedef attn_unit<HD, KV, HOW == FEW ? 1 : 4> unit;
    static constexpr int BYTES = HOW == DIRECT ? unit::BYTES_DIRECT : unit::BYTES;
    static __device__ __forceinline__ unit make(const attn_prefix& a, unsigned char* lds, attn_info* wi) {
        return unit(a, (_Float16*)lds + (HOW == FEW ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * unit::PART : 0), wi);
    }
};

// Block b of the prefix's.  Blocks are dealt round-robin to the 8 XCDs: each takes a contiguous run of them, so
// that row tiles that read the same keys share an L2.
template <int HD, typename KV, int HOW>
__device__ __forceinline__ void attn_prefix_block(const attn_prefix& a, unsigned char* lds, attn_info* wi) {
    typedef attn_how<HD, KV, HOW> how;
    const int xcd = blockIdx.x % 8, b = xcd * (a.nbp / 8) + min(xcd, a.nbp % 8) + blockIdx.x / 8;
    int at = b * a.run;
    const int end = min(at + a.run, a.NKV * a.MTp * a.stages);
    auto u = how::make(a, lds, wi);
    u.row = (int)a.kp_row;
    u.own = false;
    while (at < end) {
        const int unit = at / a.stages, t = at - unit * a.stages, g = unit / a.MTp, mt = unit % a.MTp;
        const int n = min(a.stages - t, end - at);
        u.K = (const KV*)a.kp + g * a.kp_head;
        u.V = (const KV*)a.vp + g * a.kp_head;
        u.k0 = t * a.step;
        u.k1 = (int)min((long long)a.P, (long long)(t + n) * a.step);
        u.begin(g, 0, a.R * (a.NH / a.NKV), mt * how::unit::ROWS, 0, 0);
        bool odd;
        if constexpr (HOW == DIRECT) {
            typename how::unit::source x;
            if constexpr (how::unit::NP == 1) {
                x = {(const _Float16*)u.K, (const _Float16*)u.V, 0, (int)a.kp_row, nullptr};
            } else {
                // attn_cut's: K's pieces, V's pieces, each [piece][head][key][HD]
                const long long piece = (long long)a.NKV * a.P * HD;
                const _Float16* const k = a.cut + (long long)g * a.P * HD;
                x = {k, k + 2 * piece, piece, HD, a.scales + (long long)g * ((a.P + 31) / 32) * 4};
            }
            odd = u.run_direct(x);
        } else {
            odd = u.run_staged();
        }
        u.finish(b - unit * a.stages / a.run, odd ? HOW == DIRECT ? 3 : 1 : 0);
        at += n;
        __syncthreads();
    }
}
// Block i of the own keys'.
template <int HD, typename KV, int HOW>
__device__ __forceinline__ void attn_own_block(const attn_prefix& a, int i, unsigned char* lds, attn_info* wi) {
    typedef attn_how<HD, KV, HOW> how;
    const int G = a.NH / a.NKV, mt = i % a.MTs;
    i /= a.MTs;
    const int ss = i % a.Ss;
    i /= a.Ss;
    const int g = i % a.NKV;
    seq_keys k;
    k.read(a, i / a.NKV);
    auto u = how::make(a, lds, wi);
    u.row = (int)a.ks_row;
    u.own = true;
    u.K = (const KV*)a.ks + k.first * a.ks_row + g * a.ks_head;
    u.V = (const KV*)a.vs + k.first * a.ks_row + g * a.ks_head;
    for (int v0 = mt * how::unit::ROWS; v0 < k.nq * G; v0 += a.MTs * how::unit::ROWS) {
        k.range(a, ss, v0, G, u.k0, u.k1);
        u.begin(g, k.q0, k.nq * G, v0, k.len, k.nq);
        bool odd = false;
        if (u.k0 >= u.k1) {
            u.clear();
        } else {
            if constexpr (HOW == DIRECT) odd = u.run_direct({(const _Float16*)u.K, (const _Float16*)u.V, 0, (int)a.ks_row, nullptr});
            else odd = u.run_staged();
        }
        u.finish(a.Sp + ss, odd ? 1 : 0);
        __syncthreads();
    }
}
// One launch: the prefix's blocks, then the own keys'.
template <int HD, typename KV, int PRE, int OWN>
__device__ __forceinline__ void attn_part(const attn_prefix& a) {
    constexpr int BP = attn_how<HD, KV, PRE>::BYTES, BO = attn_how<HD, KV, OWN>::BYTES;
    __shared__ __attribute__((aligned(1024))) unsigned char lds[BP > BO ? BP : BO];
    __shared__ attn_info wi[2];
    if ((int)blockIdx.x < a.nbp) attn_prefix_block<HD, KV, PRE>(a, lds, wi);
    else attn_own_block<HD, KV, OWN>(a, blockIdx.x - a.nbp, lds, wi);
}

// The prefix's fp32 K and V as two fp16 pieces each, with their scales, for the blocks of 128 rows: worth its
// way through memory and the launch where many of them read each key (the launcher's rule; 34080 rows and heads over 3001
// keys 113 us in all, 136 without).  A wave takes 32 keys; keys past the end are not written.
template <int HD>
__device__ __forceinline__ void attn_cut(const attn_prefix& a, int block) {
    typedef attn_unit<HD, float, 4> unit;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), grps = (a.P + 31) / 32, i = block * 4 + wave;
    const int g = i / grps, key = 32 * (i - g * grps);
    if (g >= a.NKV) return;
    unit u(a, nullptr, nullptr);
    u.own = false;
    u.row = (int)a.kp_row;
    u.k1 = a.P;
    const long long piece = (long long)a.NKV * a.P * HD;
    bool odd[2] = {false, false};
    int ex[2];
    typename unit::block b[2][2];
#pragma unroll
    for (int n = 0; n < 4; n++) u.load(b[n / 2][n % 2], (const float*)pick(n < 2, a.kp, a.vp) + g * a.kp_head, key + 16 * (n % 2));
#pragma unroll
    for (int p = 0; p < 2; p++) {
        u.trim(b[p][0], key);
        u.trim(b[p][1], key + 16);
        ex[p] = p ? u.template survey<true>(b[p], key, odd[p]) : u.template survey<false>(b[p], key, odd[p]);
        const float up = pow2(-ex[p]);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            typedef _Float16 part __attribute__((ext_vector_type(unit::DW)));
            const int at = key + 16 * (j / 4) + 4 * u.kq + j % 4;
            part hi, lo;
#pragma unroll
            for (int e = 0; e < unit::DW; e += 2) {
                f16x2 x, y;
                split2(b[p][j / 4].v[j % 4][e] * up, b[p][j / 4].v[j % 4][e + 1] * up, x, y);
                hi[e] = x[0];
                hi[e + 1] = x[1];
                lo[e] = y[0];
                lo[e + 1] = y[1];
            }
            if (at >= a.P) continue;
            _Float16* to = a.cut + p * 2 * piece + ((long long)g * a.P + at) * HD + u.dq * unit::DW;
            *reinterpret_cast<part*>(to) = hi;
            *reinterpret_cast<part*>(to + piece) = lo;
        }
    }
    if (u.lane == 0) *reinterpret_cast<i32x4*>(a.scales + 4ll * i) = i32x4{ex[0], ex[1], odd[0] | odd[1], 0};
}

// ... in one launch with the own keys' blocks, which come first.
template <int HD, int OWN>
__device__ __forceinline__ void attn_cut_own(const attn_prefix& a) {
    __shared__ __attribute__((aligned(1024))) unsigned char lds[attn_how<HD, float, OWN>::BYTES];
    __shared__ attn_info wi[2];
    if ((int)blockIdx.x < a.nbs) attn_own_block<HD, float, OWN>(a, blockIdx.x, lds, wi);
    else attn_cut<HD>(a, blockIdx.x - a.nbs);
}
template <int HD>
__device__ __forceinline__ void attn_cut_prefix(const attn_prefix& a) {
    __shared__ __attribute__((aligned(1024))) unsigned char lds[attn_how<HD, float, DIRECT>::BYTES];
    attn_prefix_block<HD, float, DIRECT>(a, lds, nullptr);
}

// Keys that the split's block left out, 32 at a time, of those that row r, head hd sees: on the vector ALUs in
// fp32, added to (m, l, o) by the whole wave, a key a lane for the scores, then a dim (HD 128: two) a lane.  o is the
// values' average so far, not their sum, which may leave fp32 where they do not (32 keys round it once more).  Surveys as
// the block made them (mark 1), or as attn_cut did (3); mark 2: every key.  ps: 64 floats of the wave.
template <int HD, typename KV>
__device__ void odd_tiles(const attn_prefix& a, int r, int hd, int s, int mark, float* ps, float& m, float& l,
                          float (&o)[HD > 64 ? 2 : 1]) {
    typedef attn_unit<HD, KV, 1> unit;
    const int G = a.NH / a.NKV, g = hd / G;
    unit u(a, nullptr, nullptr);
    int first = 0, k0, seen;
    u.own = s >= a.Sp;
    if (u.own) {
        int lo = 0, hi = a.B;                              // q_start[lo] <= r < q_start[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (a.q_start[mid] <= r) lo = mid;
            else hi = mid;
        }
        seq_keys k;
        k.read(a, lo);
        first = k.first;
        const int v = (r - k.q0) * G + hd - g * G, rows = a.wide_s ? 128 : 32;
        k.range(a, s - a.Sp, v / rows * rows, G, k0, u.k1);
        seen = min(max(k.len - k.nq + (r - k.q0) + 1, 0), min(k.len, u.k1));
    } else {
        const int rows = a.wide_p ? 128 : 32, unit = g * a.MTp + (r * G + hd - g * G) / rows;
        const int x = unit * a.stages, b = x / a.run + s;
        k0 = (max(b * a.run, x) - x) * a.step;
        seen = u.k1 = (int)min((long long)a.P, (long long)(min((b + 1) * a.run, x + a.stages) - x) * a.step);
    }
    const long long row = pick(u.own, a.ks_row, a.kp_row), head = pick(u.own, a.ks_head, a.kp_head);
    u.row = (int)row;
    u.K = (const KV*)pick(u.own, a.ks, a.kp) + first * row + g * head;
    u.V = (const KV*)pick(u.own, a.vs, a.vp) + first * row + g * head;
    const float* q = (const float*)a.q + r * a.q_row + hd * a.q_head;
    const int lane = u.lane;
    for (int key = k0; key < seen; key += 32) {
        bool odd = mark == 2, is;
        if (mark == 1) {
            for (int e = 0; e < 32; e += 16) {
                typename unit::block b[1];
                u.load(b[0], u.K, key + e);
                u.trim(b[0], key + e);
                u.template survey<false>(b, key + e, is);
                odd |= is;
                u.load(b[0], u.V, key + e);
                u.trim(b[0], key + e);
                u.template survey<true>(b, key + e, is);
                odd |= is;
            }
        } else if (mark == 3) {
            const int grps = (a.P + 31) / 32;
            odd = a.scales[4ll * (g * grps + key / 32) + 2] != 0;
        }
        if (!odd) continue;
        const int c = min(32, seen - key);
        const KV* kr = u.K + (long long)(key + min(lane, c - 1)) * row;
        float x = 0.0f;
        for (int d = 0; d < HD; d++) x = __builtin_fmaf(q[d], (float)kr[d], x);
        x = lane < c ? x * (a.scale * kLog2e) : -INFINITY;
        const float mn = fmaxf(m, sgpu_wave_max(x)), base = mn == -INFINITY ? 0.0f : mn;
        const float al = __builtin_amdgcn_exp2f(m - base), p = __builtin_amdgcn_exp2f(x - base);
        const float ln = __builtin_fmaf(l, al, sgpu_wave_sum(p)), part = ln == 0.0f ? 0.0f : 1.0f / ln;
        const float keep = l * al * part;
        m = mn;
        l = ln;
        ps[lane] = p * part;
        lds_sync();
#pragma unroll
        for (int e = 0; e < (HD > 64 ? 2 : 1); e++) {
            const int d = min(lane + 64 * e, HD - 1);
            o[e] *= keep;
            for (int j = 0; j < c; j++) o[e] = __builtin_fmaf(ps[j], (float)u.V[(long long)(key + j) * row + d], o[e]);
        }
        lds_sync();
    }
}

// The splits of each row and head joined: by a wave (64 / T splits side by side, HD = 4 T dims) where there are
// more than 8 splits, else by T lanes.  U records a lane are on their way at once (16: 63 splits of 56 rows and heads
// 4.8 us, 9.0 with 8; but 9 of 1536 5.3 us, 4.1 with 8).  Bound: the records' way through memory (1536 rows and
// heads of 128 dims by 33 splits, 26 MB: 9 us; 34080 of 64 dims by 3 to 4: 13.5 us), below that two rounds of loads.
template <int HD, typename KV, bool MANY>
__device__ __forceinline__ void attn_join(const attn_prefix& a) {
    constexpr int T = HD / 4, TEAM = MANY ? 64 : T, N = TEAM / T, RD = HD > 64 ? 2 : 1;
    __shared__ __attribute__((aligned(16))) float odd_o[4][HD], ps[4][64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, part = lane % TEAM / T;
    const int n = a.R * a.NH, G = a.NH / a.NKV, t = (blockIdx.x * 256 + threadIdx.x) / TEAM, d = (lane % T) * 4;
    const int r = min(t, n - 1) / a.NH, hd = min(t, n - 1) - r * a.NH;
    const bool live = t < n && r >= a.q_start[0] && r < a.q_start[a.B];
    int cnt = 0;                                                   // splits of the prefix
    if (a.nbp > 0) {
        const int x = (hd / G * a.MTp + (r * G + hd % G) / (a.wide_p ? 128 : 32)) * a.stages;
        cnt = (x + a.stages - 1) / a.run - x / a.run + 1;
    }
    const int S = live ? cnt + a.Ss : 0;
    const sgpu_f32x4* ml = reinterpret_cast<const sgpu_f32x4*>(a.pml);
    auto rec = [&](int s, int at) __attribute__((always_inline)) { return (size_t)(s < cnt ? s : a.Sp + s - cnt) * n + at; };
    float M = -INFINITY, L = 0.0f;
    sgpu_f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
    bool odd = false;
    auto splits = [&](auto at_once) __attribute__((always_inline)) {
        constexpr int U = decltype(at_once)::value;
        for (int s0 = 0; __any(s0 < S); s0 += U * N) {                 // (S differs between a wave's rows)
            sgpu_f32x4 y[U], v[U];
#pragma unroll
            for (int k = 0; k < U; k++) {
                const int s = s0 + k * N + part;
                y[k] = s < S ? ml[rec(s, t)] : sgpu_f32x4{-INFINITY, 0.0f, 0.0f, 0.0f};
                v[k] = s < S ? *reinterpret_cast<const sgpu_f32x4*>(a.po + rec(s, t) * HD + d) : sgpu_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
            float mn = M;
#pragma unroll
            for (int k = 0; k < U; k++) {
                odd |= y[k][2] != 0.0f;
                if (y[k][2] == 2.0f || y[k][1] == 0.0f) y[k] = sgpu_f32x4{-INFINITY, 0.0f, 0.0f, 0.0f};    // not to be used
                mn = fmaxf(mn, y[k][0]);
            }
            const float base = mn == -INFINITY ? 0.0f : mn, al = __builtin_amdgcn_exp2f(M - base);
            M = mn;
            L *= al;
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] *= al;
#pragma unroll
            for (int k = 0; k < U; k++) {
                const float w = __builtin_amdgcn_exp2f(y[k][0] - base);
                L = __builtin_fmaf(y[k][1], w, L);
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] = y[k][1] == 0.0f ? x[e] : __builtin_fmaf(v[k][e], w, x[e]);
            }
        }
    };
    if (!MANY) splits(std::integral_constant<int, 4>());
    else if (a.Sp + a.Ss <= 8 * N) splits(std::integral_constant<int, 8>());
    else splits(std::integral_constant<int, 16>());
    auto merge = [&](float m, float l, const sgpu_f32x4& v) __attribute__((always_inline)) {
        const float mn = fmaxf(M, m), base = mn == -INFINITY ? 0.0f : mn;
        const float al = __builtin_amdgcn_exp2f(M - base), be = __builtin_amdgcn_exp2f(m - base);
        M = mn;
        L = L * al + l * be;
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = l == 0.0f ? x[e] * al : __builtin_fmaf(v[e], be, x[e] * al);
    };
#pragma unroll
    for (int o = T; o < TEAM; o *= 2) {                            // the parts of a row, both sides alike
        const sgpu_f32x4 v = {__shfl_xor(x[0], o), __shfl_xor(x[1], o), __shfl_xor(x[2], o), __shfl_xor(x[3], o)};
        const float m2 = __shfl_xor(M, o), l2 = __shfl_xor(L, o);
        const bool first = (lane & o) == 0;                        // the same order of the sum on both
        if (first) {
            merge(m2, l2, v);
        } else {
            const sgpu_f32x4 mine = x;
            const float m1 = M, l1 = L;
            x = v;
            M = m2;
            L = l2;
            merge(m1, l1, mine);
        }
        odd |= __shfl_xor((int)odd, o) != 0;
    }
    if (__any(odd)) {                                              // rare: the wave takes what the blocks left out, row by row
        for (int j = 0; j < 64; j += TEAM) {
            if (!__builtin_amdgcn_readlane((int)odd, j)) continue;
            const int rj = __builtin_amdgcn_readlane(r, j), hj = __builtin_amdgcn_readlane(hd, j), tj = __builtin_amdgcn_readlane(t, j);
            const int sj = __builtin_amdgcn_readlane(S, j), cj = __builtin_amdgcn_readlane(cnt, j);
            float om = -INFINITY, ol = 0.0f, o[RD];
#pragma unroll
            for (int e = 0; e < RD; e++) o[e] = 0.0f;
            for (int s = 0; s < sj; s++) {
                const int at = s < cj ? s : a.Sp + s - cj;
                const float mark = ml[(size_t)at * n + tj][2];
                if (mark != 0.0f) odd_tiles<HD, KV>(a, rj, hj, at, (int)mark, ps[wave], om, ol, o);
            }
#pragma unroll
            for (int e = 0; e < RD; e++)
                if (lane + 64 * e < HD) odd_o[wave][lane + 64 * e] = o[e];
            lds_sync();
            if (lane / TEAM == j / TEAM) {                         // of averages, as odd_tiles holds them
                const sgpu_f32x4 v = *reinterpret_cast<const sgpu_f32x4*>(&odd_o[wave][d]);
                const float mn = fmaxf(M, om), base = mn == -INFINITY ? 0.0f : mn;
                const float ex = __builtin_amdgcn_exp2f(M - base), lv = ol * __builtin_amdgcn_exp2f(om - base);
                const float part = 1.0f / __builtin_fmaf(L, ex, lv);
                const float wx = L == 0.0f ? 0.0f : ex * part, wv = lv * part;
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] = ol == 0.0f ? x[e] * wx : __builtin_fmaf(v[e], wv, x[e] * wx);
                L = L == 0.0f && ol == 0.0f ? 0.0f : 1.0f;
            }
            lds_sync();
        }
    }
    if (!live || part != 0) return;
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] = L == 0.0f ? 0.0f : x[e] / L;
    *reinterpret_cast<sgpu_f32x4*>(a.out + r * a.out_row + hd * a.out_head + d) = x;
}

}  // namespace

#define SGPU_ROPE(NAME, O, INTER, VEC)                                                                                \
    extern "C" __global__ void __launch_bounds__(256) sgpu_rope_rows_##NAME(                                          \
        const float* x, long long xs, O* y, long long ys, const int* __restrict__ pos, int pos0,                      \
        const double* __restrict__ turns, int rot, float mscale, int T, int H, int HD, int tb, int same) {            \
        rope_rows<O, INTER, VEC>(x, xs, y, ys, pos, pos0, turns, rot, mscale, T, H, HD, tb, same);                    \
    }
SGPU_ROPE(half_f32, float, false, false)
SGPU_ROPE(half_f16, _Float16, false, false)
SGPU_ROPE(half_v4_f32, float, false, true)
SGPU_ROPE(half_v4_f16, _Float16, false, true)
SGPU_ROPE(inter_f32, float, true, false)
SGPU_ROPE(inter_f16, _Float16, true, false)
SGPU_ROPE(inter_v4_f32, float, true, true)
SGPU_ROPE(inter_v4_f16, _Float16, true, true)

#define SGPU_LP(NAME, X)                                                                                              \
    extern "C" __global__ void __launch_bounds__(256) sgpu_lp_part_##NAME(                                            \
        const X* __restrict__ x, long long xs, int V, int C, int len, int k, float* __restrict__ part,                \
        unsigned long long* __restrict__ keys) {                                                                      \
        lp_part<X>(x, xs, V, C, len, k, part, keys);                                                                  \
    }                                                                                                                 \
    extern "C" __global__ void __launch_bounds__(64) sgpu_lp_join_##NAME(                                             \
        const X* __restrict__ x, long long xs, int V, int C, const int* __restrict__ tok, int nt,                     \
        float* __restrict__ logp, float* __restrict__ entropy, int k, float* __restrict__ top_logp,                   \
        int* __restrict__ top_id, const float* __restrict__ part, const unsigned long long* __restrict__ keys) {      \
        lp_join<X>(x, xs, V, C, tok, nt, logp, entropy, k, top_logp, top_id, part, keys);                             \
    }
SGPU_LP(f32, float)
SGPU_LP(f16, _Float16)

#define SGPU_ATTN_KERNEL(HD, WAVES, NAME, BODY)                                                                       \
    extern "C" __global__ void __launch_bounds__(256, WAVES) sgpu_attn_##NAME##_##HD(attn_prefix a) { BODY; }
#define SGPU_ATTN(HD)                                                                                                 \
    SGPU_ATTN_KERNEL(HD, (HD) <= 64 ? 2 : 1, few_f32, (attn_part<HD, float, FEW, FEW>(a)))                            \
    SGPU_ATTN_KERNEL(HD, (HD) <= 64 ? 2 : 1, few_f16, (attn_part<HD, _Float16, FEW, FEW>(a)))                         \
    SGPU_ATTN_KERNEL(HD, (HD) <= 64 ? 2 : 1, step_f32, (attn_part<HD, float, ROWS, FEW>(a)))                          \
    SGPU_ATTN_KERNEL(HD, (HD) <= 64 ? 2 : 1, rows_f32, (attn_part<HD, float, ROWS, ROWS>(a)))                         \
    SGPU_ATTN_KERNEL(HD, 2, rows_f16, (attn_part<HD, _Float16, DIRECT, DIRECT>(a)))                                   \
    SGPU_ATTN_KERNEL(HD, (HD) <= 64 ? 2 : 1, cut_step, (attn_cut_own<HD, FEW>(a)))                                    \
    SGPU_ATTN_KERNEL(HD, (HD) <= 64 ? 2 : 1, cut_rows, (attn_cut_own<HD, ROWS>(a)))                                   \
    SGPU_ATTN_KERNEL(HD, (HD) <= 64 ? 3 : 2, cut_prefix, (attn_cut_prefix<HD>(a)))                                    \
    SGPU_ATTN_KERNEL(HD, 1, join_few_f32, (attn_join<HD, float, false>(a)))                                           \
    SGPU_ATTN_KERNEL(HD, 1, join_few_f16, (attn_join<HD, _Float16, false>(a)))                                        \
    SGPU_ATTN_KERNEL(HD, 1, join_many_f32, (attn_join<HD, float, true>(a)))                                           \
    SGPU_ATTN_KERNEL(HD, 1, join_many_f16, (attn_join<HD, _Float16, true>(a)))
SGPU_ATTN(32)
SGPU_ATTN(64)
SGPU_ATTN(128)
