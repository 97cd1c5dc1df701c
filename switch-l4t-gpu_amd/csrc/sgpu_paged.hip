// sgpu_paged.hip -- what a host that serves several requests from one paged cache, and checks tokens drafted
// ahead, needs beside the decode engines' own kernels (gfx950):
//   sgpu_heads_*    each head's norm and rotation, into rows or into the pages of a cache
//   sgpu_tree_*     attention of new rows over their sequence's pages, with a tree's mask over the new ones
//   sgpu_logits_*   penalties, biases and a grammar's mask on logits
// fp16 values here are IEEE ones, as in sgpu_score.hip.
#include <type_traits>

#include "sgpu_rows.h"

// What the launchers pass by value.
struct paged_heads {
    const float *q, *k, *v;               // row t, head h at t * row + h * HD
    void *yq, *yk, *yv;                   // rows of yq, yk; pages: yk, yv are the cache's
    const float *wq, *wk;
    const int* pos;
    const double* turns;
    const int *table, *len, *q_start;
    long long q_row, k_row, v_row, yq_row, yk_row, table_row, page_stride, kv_row, kv_head;
    int pos0, rot, neighbours;
    float mscale, eps;
    double per;                           // 1 / HD
    int T, NH, NKV, HD, tb, team;         // rows a block, log2 of a head's lanes
    int pages, page, table_pages, B;
};
struct paged_tree {
    const void *k, *v;
    const float* q;
    float* out;
    const int* table;
    const uint32_t* mask;
    float *po, *pml;                      // records of partial units, two a block: outputs; (max, sum)
    int* desc;                            // of each row and head: (first block << 8 | row of the tile, records; 0: nothing to join)
    long long page_stride, kv_row, kv_head, table_row, q_row, q_head, out_row, out_head, mask_row;
    int pages, page, table_pages, NH;
    float scale;
    int MT, shift;                        // row tiles of a sequence and KV head (NB 0); log2 of page (-1: none)
    int halves;                           // 16 aligned tokens lie on one page, 64 of their rows within 2^31 bytes
};
// What a block needs first: as arguments of their own, which are in its registers when it starts.
struct tree_front {
    const int *q_start, *len;
    int B, R, NKV, G, room;               // G = NH / NKV; room: tokens of a table's row
    int NB;                               // blocks the steps are dealt to; 0: a block a row tile
    int start;                            // what a unit's beginning costs a block beside its steps, in steps (0: a block a step)
    int magic;                            // ceil(2^32 / G) where multiplying by it divides row numbers by G, else 0
    __device__ __forceinline__ int row_of(int v) const { return magic ? (int)__umulhi((uint32_t)v, (uint32_t)magic) : G == 1 ? v : v / G; }
};
struct paged_logits {
    const void* x;
    void* y;
    const int *tok, *span, *bias_id, *bias_span;
    const float *rep, *freq, *pres, *bias;
    const uint32_t* allow;
    long long x_row, y_row, allow_row;
    int rows, V, n_tok, n_bias, C, groups;        // C: chunks of a row, dealt to `groups` blocks
};

namespace {

typedef int i32x2 __attribute__((ext_vector_type(2)));
constexpr float kLog2e = 1.44269504088896340736f;

// ---- the batch ----
// The sequence of row r, the last b with q_start[b] <= r, by the whole wave (64 starts at a time); -1 for rows
// of none.
__device__ __forceinline__ int sequence_of(const int* __restrict__ q_start, int B, int r) {
    if (r < q_start[0] || r >= q_start[B]) return -1;
    const int lane = threadIdx.x & 63;
    int lo = 0, n = B;
    while (n > 1) {
        const int step = (n + 63) / 64, at = lane * step;
        const int c = max(__popcll(__ballot(at < n && q_start[lo + min(at, n - 1)] <= r)), 1) - 1;
        lo += c * step;
        n = min(step, n - c * step);
    }
    return lo;
}
// The page of token `at` of sequence b; -1 where its table has none.
template <typename A> __device__ __forceinline__ int page_of(const A& a, int b, long long at) {
    if (at < 0 || at >= (long long)a.table_pages * a.page) return -1;
    const int p = a.table[b * a.table_row + (int)at / a.page];
    return p >= 0 && p < a.pages ? p : -1;
}

// ---- heads: norm and rotation ----
constexpr int kAngles = 2048;             // (cos, sin) pairs a block holds: its rows by rot / 2
constexpr int kHeadRows = 64;             // the most rows of a block

// 1 / sqrt(x): the 64-bit approximation and one step of Newton's method (2^-46 or better); 0 of infinity, which the step
// would make a NaN of (x infinite beside finite values: theirs are 0).
__device__ __forceinline__ double inv_sqrt(double x) {
    const double y = __builtin_amdgcn_rsq(x);
    return y == 0.0 ? y : y * (1.5 - 0.5 * x * y * y);
}
// r = f g as fp32 factors, mostly f = r and g = 1.  (The inverse of a root mean square below 2^-128 is no fp32 number, that of
// one above 2^126 has few digits: both get half of its power of two.  x r is of order 1 all the same.  A branch for it
// measured the same and took more registers.)
__device__ __forceinline__ float fp32_factors(double r, float& g) {
    const int k = __builtin_amdgcn_frexp_exp(r), half = k > -126 && k < 128 ? 0 : k / 2;
    g = __builtin_amdgcn_ldexpf(1.0f, half);
    return (float)__builtin_amdgcn_ldexp(r, -half);
}
// The sum of `lanes` neighbouring lanes (a power of 2, the same for all), in all of them.
__device__ __forceinline__ double lanes_sum(double s, int lanes) {
    auto add = [&](auto ctrl) __attribute__((always_inline)) {
        const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(s), decltype(ctrl)::value, 0xf, 0xf, true);
        const int hi = __builtin_amdgcn_update_dpp(0, __double2hiint(s), decltype(ctrl)::value, 0xf, 0xf, true);
        s += __hiloint2double(hi, lo);
    };
    if (lanes > 1) add(std::integral_constant<int, 0xB1>());       // quads 1 0 3 2
    if (lanes > 2) add(std::integral_constant<int, 0x4E>());       // quads 2 3 0 1
    if (lanes > 4) add(std::integral_constant<int, 0x141>());      // eights mirrored
    if (lanes > 8) add(std::integral_constant<int, 0x140>());      // rows of 16 mirrored
    if (lanes > 16) s += __shfl_xor(s, 16);
    if (lanes > 32) s += __shfl_xor(s, 32);
    return s;
}

__device__ __forceinline__ sgpu_f32x4 neighbours_turned(sgpu_f32x4 y, const float* tab) {      // two pairs
    const sgpu_f32x4 k = *reinterpret_cast<const sgpu_f32x4*>(tab);
    return sgpu_f32x4{y[0] * k[0] - y[1] * k[1], y[0] * k[1] + y[1] * k[0], y[2] * k[2] - y[3] * k[3], y[2] * k[3] + y[3] * k[2]};
}
template <bool ONCE, typename O> __device__ __forceinline__ void put_quad(O* p, sgpu_f32x4 v) {
    typedef O quad __attribute__((ext_vector_type(4)));
    const quad y = __builtin_convertvector(v, quad);
    if constexpr (ONCE) __builtin_nontemporal_store(y, reinterpret_cast<quad*>(p));
    else *reinterpret_cast<quad*>(p) = y;
}

// Rows t of q (NH heads), k (NKV) and, into pages, v (NKV): y = rot(x * w / sqrt(mean x^2 + eps)), the norm where
// there are weights, its squares summed in 64 bits (no value's square leaves them); v as it is.  Pair i of a head is (i, i + rot/2),
// or (2i, 2i+1), and turns by turns[i] per position.  PAGED: row t is token len[b] + i of its sequence b, k and v go to
// its place in the pages (rows without one are left out), and rows of no sequence are left as they were.
// A block takes tb rows: their places and angles once into LDS, then every head reads them.  VEC: 2^team lanes a
// head, eight values each (a pair's both sides in one lane); otherwise a wave a head, a pair or a value a lane.  ONCE: read and
// written past the caches' usual order.
// In place is fine: a head's values are all read before the first is written.
// Bound by memory: 4099 rows of 40 heads of 128 to fp16 (126 MB) 25.8 us, 4.9 TB/s, as a large copy; 5500 rows appended to fp16 pages
// (247 MB) 48.8 us, 5.1 TB/s; one row 2.6 us, the launch.  Sums over lanes by DPP instead of shuffles 31 -> 28 us of the
// first, past the caches' order 29 -> 26.
template <typename QO, typename KO, bool PAGED, bool VEC, bool ONCE>
__device__ __forceinline__ void heads(const paged_heads& a) {
    __shared__ __attribute__((aligned(16))) float table[2 * kAngles];
    __shared__ long long places[kHeadRows], positions[kHeadRows];  // where in the pages: -1 nowhere, -2 no row
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int half = a.rot / 2, HD = a.HD, H = a.NH + a.NKV + (PAGED ? a.NKV : 0);
    for (int t0 = blockIdx.x * a.tb; t0 < a.T; t0 += gridDim.x * a.tb) {
        const int n = min(a.tb, a.T - t0);
        if constexpr (PAGED) {
            for (int t = wave; t < n; t += 4) {
                const int r = t0 + t, b = sequence_of(a.q_start, a.B, r);
                long long place = -2, p = 0;
                if (b >= 0) {
                    const long long at = (long long)a.len[b] + (r - a.q_start[b]);
                    const int page = page_of(a, b, at);
                    place = page < 0 ? -1 : page * a.page_stride + at % a.page * a.kv_row;
                    p = a.pos ? a.pos[r] : at;
                }
                if (lane == 0) {
                    places[t] = place;
                    positions[t] = p;
                }
            }
            __syncthreads();
        }
        for (int i = tid; i < n * half; i += 256) {
            const int t = i / half;
            const long long p = PAGED ? positions[t] : (long long)a.pos0 + (a.pos ? a.pos[t0 + t] : t0 + t);
            float s, c;
            sincos_turns((double)p * a.turns[i - t * half], s, c);
            table[2 * i] = c * a.mscale;
            table[2 * i + 1] = s * a.mscale;
        }
        __syncthreads();
        const int lanes = VEC ? 1 << a.team : 64;
        for (int i = tid; i < n * H * lanes; i += 256) {
            const int e = i & (lanes - 1), th = VEC ? i >> a.team : i >> 6, h = th % H, t = th / H;
            const int kind = h < a.NH ? 0 : h < a.NH + a.NKV ? 1 : 2, hh = h - (kind == 0 ? 0 : kind == 1 ? a.NH : a.NH + a.NKV);
            const float* const x = kind == 0 ? a.q + (t0 + t) * a.q_row + (long long)hh * HD
                                   : kind == 1 ? a.k + (t0 + t) * a.k_row + (long long)hh * HD
                                               : a.v + (t0 + t) * a.v_row + (long long)hh * HD;
            QO* const yq = (QO*)a.yq + (t0 + t) * a.yq_row + (long long)hh * HD;
            KO* yk;
            if constexpr (PAGED) {
                const long long place = places[t];
                if (place == -2 || (kind > 0 && place < 0)) continue;
                yk = (KO*)(kind == 1 ? a.yk : a.yv) + place + hh * a.kv_head;
            } else {
                yk = (KO*)a.yk + (t0 + t) * a.yk_row + (long long)hh * HD;
            }
            const float* const w = kind == 0 ? a.wq : kind == 1 ? a.wk : nullptr;
            const float* const tab = table + 2 * t * half;
            const int rot = kind < 2 ? a.rot : 0;
            if constexpr (VEC) {
                // lane e's two quads: both sides of pairs that lie apart; neighbouring lanes' quads lie side by side
                const bool live = e < HD / 8;
                const int split = a.neighbours ? 0 : rot / 8;      // lanes with such pairs
                const bool apart = e < split;
                const int d0 = 4 * (apart ? e : split + e), d1 = 4 * (apart ? split + e : HD / 8 + e);
                sgpu_f32x4 u = {}, v = {};
                if (live) {
                    const sgpu_f32x4 *const p0 = reinterpret_cast<const sgpu_f32x4*>(x + d0), *const p1 = reinterpret_cast<const sgpu_f32x4*>(x + d1);
                    u = ONCE ? sgpu_ldnt(p0) : *p0;
                    v = ONCE ? sgpu_ldnt(p1) : *p1;
                }
                if (w) {
                    sgpu_f32x4 p = {}, q = {};
                    if (live) {
                        p = *reinterpret_cast<const sgpu_f32x4*>(w + d0);
                        q = *reinterpret_cast<const sgpu_f32x4*>(w + d1);
                    }
                    double s = 0.0;
#pragma unroll
                    for (int j = 0; j < 4; j++) s = __builtin_fma((double)v[j], (double)v[j], __builtin_fma((double)u[j], (double)u[j], s));
                    float g;
                    const float f = fp32_factors(inv_sqrt(__builtin_fma(lanes_sum(s, lanes), a.per, (double)a.eps)), g);
                    u = u * f * g * p;
                    v = v * f * g * q;
                }
                if (!live) continue;
                if (apart) {
                    const sgpu_f32x4 k0 = *reinterpret_cast<const sgpu_f32x4*>(tab + 2 * d0), k1 = *reinterpret_cast<const sgpu_f32x4*>(tab + 2 * d0 + 4);
                    const sgpu_f32x4 c = {k0[0], k0[2], k1[0], k1[2]}, sn = {k0[1], k0[3], k1[1], k1[3]}, p = u;
                    u = p * c - v * sn;
                    v = p * sn + v * c;
                } else if (a.neighbours) {
                    if (d0 < rot) u = neighbours_turned(u, tab + d0);
                    if (d1 < rot) v = neighbours_turned(v, tab + d1);
                }
                if (kind == 0) {
                    put_quad<ONCE>(yq + d0, u);
                    put_quad<ONCE>(yq + d1, v);
                } else {
                    put_quad<ONCE>(yk + d0, u);
                    put_quad<ONCE>(yk + d1, v);
                }
            } else {
                float f = 1.0f, g = 1.0f;
                if (w) {
                    double s = 0.0;
                    for (int d = e; d < HD; d += 64) s += (double)x[d] * x[d];
                    f = fp32_factors(inv_sqrt(__builtin_fma(lanes_sum(s, 64), a.per, (double)a.eps)), g);
                }
                auto at = [&](int d) __attribute__((always_inline)) { return w ? x[d] * f * g * w[d] : x[d]; };
                auto put = [&](int d, float y) __attribute__((always_inline)) {
                    if (kind == 0) yq[d] = (QO)y;
                    else yk[d] = (KO)y;
                };
                for (int p = e; p < rot / 2; p += 64) {
                    const int i0 = a.neighbours ? 2 * p : p, i1 = a.neighbours ? 2 * p + 1 : half + p;
                    const float u = at(i0), v = at(i1), c = tab[2 * p], s = tab[2 * p + 1];
                    put(i0, u * c - v * s);
                    put(i1, u * s + v * c);
                }
                for (int d = rot + e; d < HD; d += 64) put(d, at(d));
            }
        }
        __syncthreads();                              // the tables are the next rows'
    }
}

// ---- attention over pages ----
constexpr int kLeastV = -64, kMostV = 32;     // scales of V that the running sums bear beside each other (tree_unit)
// A score is a product below 2^37 (2^30 beside the largest keys, 2^120) by 2^k by 2^q scale, k and q the scales of its key and query
// row.  2^kLessK of the second goes to the third: the first two's product stays below 2^127 for every key, and where the third is
// rounded below fp32's normal range, by 2^-150, the score is off by 2^-24 at most.
constexpr int kLessK = 24;

// The largest of GROUP neighbouring lanes' numbers, in all of them.
template <int GROUP> __device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
    auto step = [&](auto ctrl) __attribute__((always_inline)) {
        const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, 0xf, 0xf, true);
        v = o > v ? o : v;
    };
    step(std::integral_constant<int, 0xB1>());                     // quads 1 0 3 2
    step(std::integral_constant<int, 0x4E>());                     // quads 2 3 0 1
    if constexpr (GROUP > 4) step(std::integral_constant<int, 0x141>());       // eights mirrored
    if constexpr (GROUP > 8) step(std::integral_constant<int, 0x140>());       // rows of 16 mirrored
    return v;
}

// Which of the 32 keys from `key` on row i sees, a bit each: those in the cache before (have), and of the new ones those of
// its mask, or up to its own.
__device__ __forceinline__ uint32_t seen_by(int key, int have, int N, int i, bool masked, const uint32_t* w, long long words) {
    const int old = have - key, j = key - have;
    if (old >= 32) return ~0u;
    uint32_t bits;
    if (!masked) {
        const int c = i - j + 1;
        bits = c >= 32 ? ~0u : c > 0 ? (1u << c) - 1 : 0;
    } else if (old > 0) {
        bits = (words > 0 ? w[0] << old : 0) | ((1u << old) - 1);
    } else {
        const int at = j / 32, s = j % 32;
        bits = at < words ? w[at] >> s : 0;
        if (s && at + 1 < words) bits |= w[at + 1] << (32 - s);
    }
    const int left = N - key;
    return left >= 32 ? bits : left > 0 ? bits & ((1u << left) - 1) : 0;
}
// ONCE: what is read by one block only, past the caches' usual order (64 ragged requests 27.9 -> 26.1 us).
template <bool ONCE, typename V> __device__ __forceinline__ V ld16(const V* p) {
    if constexpr (ONCE) return __builtin_nontemporal_load(p);
    else return *p;
}
// The exponent e that brings values of magnitude bits m below 2^15, and the largest to 2^7 or more, as x * 2^-e: a
// multiple of 8, so that most tiles have one for all keys (-120 at least: 2^-e stays a number).
__device__ __forceinline__ int row_scale(uint32_t m) { return max(((int)(m >> 23) - 134) & ~7, -120); }
template <typename KV> struct page_values;
template <> struct page_values<float> {
    static constexpr int PIECES = 2;
    struct raw { sgpu_f32x4 a, b; };                               // eight values of a key
    template <bool ONCE> static __device__ __forceinline__ raw load(const float* p) {
        return {ld16<ONCE>(reinterpret_cast<const sgpu_f32x4*>(p)), ld16<ONCE>(reinterpret_cast<const sgpu_f32x4*>(p + 4))};
    }
};
template <> struct page_values<_Float16> {
    static constexpr int PIECES = 1;
    struct raw { f16x8 a; };
    template <bool ONCE> static __device__ __forceinline__ raw load(const _Float16* p) { return {ld16<ONCE>(reinterpret_cast<const f16x8*>(p))}; }
};
template <int KT> struct key_info { float k[KT], v[KT], back[KT]; };   // 2^(scale - kLessK) of K, scale of V, 2^-scale of V

// W * WR query rows (query row, head of the group) of one sequence against keys k0 .. k1-1 of one KV head, on the fp16
// matrix cores.  Of the four waves, wave w has rows W (w % WR) .. (W: 32 or 16, by the matrix instruction) and every 4 / WR -th
// tile of 32 keys; the WR waves of a key group bring its tiles together.
//
// fp32 operands are cut into two fp16 pieces with a power of two as scale, one a query row and one a key's K and V, of
// whose four products the three larger ones are summed in fp32: 22 bits of every operand (2^-32 of the row's
// largest where that is more).  fp16 pages are one piece, exact.
// Softmax weights are cut the same way: P = 2^(x + e - M + OFF), x the score in powers of two, e the scale of the key's V,
// M the row's largest x + e so far or up to 2^LAG below it, so that O, which the matrix cores add to in place, is hardly ever
// scaled again.  The sum l of 2^(x - M + OFF) is P 2^-e before the cut.  With V's scales within kLeastV .. kMostV both
// stay normal numbers wherever they count.  A value of V past those sizes, or what is not a finite number in
// K, V or q, leaves a NaN in l or O: the wave then takes its rows and keys again on the vector ALUs (plain).
//
// Both products run transposed, so that a lane holds one row, lane h of the LR = 64 / W that do: S^T = K Q^T in quads of keys
// 4 LR n + 4 h .., O^T = V^T P^T in quads of dims 4 LR n + 4 h ..  The order of keys within a product's step is free, and
// so P is the second's B operand where the first left it; V^T comes from row-major V by LDS reads that transpose.
template <int HD, typename KV, int WR, int W> struct tree_unit {
    typedef page_values<KV> values_of;
    typedef typename values_of::raw raw;
    static constexpr int NP = values_of::PIECES, LR = 64 / W, ROWS = W * WR, WK = 4 / WR;
    static constexpr int NK = HD / (8 * LR), SQ = 8 / LR, OQ = HD / (4 * LR);    // steps of the first product, quads of scores and of dims a lane
    static constexpr int SV = W == 32 ? 1 : 2, OV = W == 32 ? HD / 32 : HD / 16; // accumulators
    typedef std::conditional_t<W == 32, f32x16, sgpu_f32x4> acc;
    static constexpr float OFF = NP == 2 ? 8.0f : 14.0f, LAG = NP == 2 ? 7.0f : 1.0f;      // P up to 2^15
    static constexpr int NC = HD / 8, GT = 64 * WR;    // chunks of a row, threads of a key group
    // Tiles of 32 keys at once, keys, chunks a thread.  Two tiles where a block's waves share them: half as many waits
    // for one another; 32 sequences with 24 drafted rows each 48.0 us with one tile, 44.9 with two.
    static constexpr int KB = WR == 4 && HD <= 64 ? 2 : 1, KT = 32 * KB, NL = 2 * KT * NC / GT;
    typedef key_info<KT> keys;
    static constexpr int TILE = KT * HD, REGION = 2 * NP * TILE, BUFS = WR == 1 ? 1 : 2;   // halves: [buffer][K, V][piece][key][HD]
    static constexpr int RPK = NC < 16 ? 16 / NC : 1;
    static constexpr int BYTES_TILES = WK * BUFS * REGION * 2, BYTES_MERGE = WK == 1 ? 0 : 4 * W * (HD + 6) * 4;
    static constexpr int BYTES = BYTES_TILES > BYTES_MERGE ? BYTES_TILES : BYTES_MERGE;

    const paged_tree& a;
    const tree_front& c;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lw = lane % W, h = lane / W;
    const int wr = wave % WR, wk = wave / WR, tg = wr * 64 + lane;
    keys* const info;                             // the key group's
    uint32_t kr, vr, kw, vw;                          // LDS addresses of this lane's reads and writes (see tile_at)
    int b, g, q0, nq, have, N, i;                     // the sequence, KV head, its rows and keys; this lane's row of it
    bool live, idle;                                  // there is such a row; the wave has none
    const float* q_at;
    const KV *K, *V;
    int qx;                                           // the row's scale: q is pieces * 2^qx
    f16x8 q[2][NK];
    acc o[OV];
    float m, l;

    // Element c of quad n of accumulators.
    template <typename A> static __device__ __forceinline__ auto get(const A& v, int n, int c) { return W == 32 ? v[n / 4][(4 * n + c) % 16] : v[n][c]; }
    template <typename A> static __device__ __forceinline__ void set(A& v, int n, int c, float x) {
        if constexpr (W == 32) v[n / 4][(4 * n + c) % 16] = x;
        else v[n][c] = x;
    }
    static __device__ __forceinline__ acc product(f16x8 x, f16x8 y, acc z) {
        if constexpr (W == 32) return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, z, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, z, 0, 0, 0);
    }
    // Over the lanes of a row.
    static __device__ __forceinline__ float row_max(float x) {
        if constexpr (LR == 4) {
            const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
            x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
        }
        return half_max(x);
    }
    static __device__ __forceinline__ float row_sum(float x) {
        if constexpr (LR == 4) {
            const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
            x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
        }
        return half_sum(x);
    }

    // Tiles lie [K, V][piece][key][HD], 16-byte chunks of a row swizzled so that 16 lanes' chunks of a column use all banks:
    // K's chunk c at c ^ (key / RPK % NC), V's bytes turned by the key's lower bits (the 8 keys by 16 dims of a
    // transposing read).  Every address is one of four of the lane, exclusive-or'd and added to by constants.
    static __device__ __forceinline__ int v_turn(int key) {
        return (HD == 32 ? 0 : HD == 64 ? 64 * (key >> 1 & 1) : 64 * (key & 3)) ^ (W == 16 ? 32 * (key >> 2 & 1) : 0);
    }
    __device__ __forceinline__ tree_unit(const paged_tree& a_, const tree_front& c_, void* lds, keys* f) : a(a_), c(c_), info(f + wk * BUFS) {
        const uint32_t base = (uint32_t)(uintptr_t)(lds_void*)lds + wk * BUFS * REGION * 2;
        const int n = lane & 15, key = 4 * h + (n >> 2), wkey = tg / NC % KT, col = tg % NC;
        kr = base + 2 * HD * lw + 16 * (h ^ (lw / RPK % NC));
        vr = base + 2 * (NP * TILE + HD * key) + (v_turn(key) ^ (W == 32 ? 32 * (lane >> 4 & 1) : 0)) + 8 * (n & 3);
        kw = base + 2 * HD * wkey + 16 * (col ^ (wkey / RPK % NC));
        vw = base + 2 * (NP * TILE + HD * wkey) + ((16 * col) ^ v_turn(wkey));
    }
    __device__ __forceinline__ void sequence(int b_, int g_, int q0_, int nq_, int have_, int N_) {
        b = b_;
        g = g_;
        q0 = q0_;
        nq = nq_;
        have = have_;
        N = N_;
        K = (const KV*)a.k + g * a.kv_head;
        V = (const KV*)a.v + g * a.kv_head;
    }
    __device__ __forceinline__ void rows(int v0) {    // rows and heads of the group from v0 on
        const int nv = nq * c.G, v = v0 + W * wr + lw, w = min(v, nv - 1);
        live = v < nv;
        idle = v0 + W * wr >= nv;
        i = c.row_of(w);
        q_at = a.q + (q0 + i) * a.q_row + (g * c.G + w - i * c.G) * a.q_head;
    }
    __device__ __forceinline__ uint32_t seen(int key) const {
        return live ? seen_by(key, have, N, i, a.mask != nullptr, a.mask + (q0 + i) * a.mask_row, a.mask_row) : 0;
    }

    // ---- pages ----
    // The page number of key tile + lane % KT (-1 past the table), and from it where the key lies.
    __device__ __forceinline__ int number(int tile) const {
        const int at = split(tile + lane % KT);
        return at < a.table_pages ? a.table[b * a.table_row + at] : -1;
    }
    __device__ __forceinline__ int split(int key) const { return a.shift >= 0 ? key >> a.shift : key / a.page; }
    struct spots {
        long long at;                                 // of key lane % KT: values from K or V; 0 where there is none
        unsigned long long valid;                     // the wave's, a bit a key
    };
    __device__ __forceinline__ spots find(int tile, int page, int k1) const {
        const int key = tile + lane % KT;
        const bool ok = page >= 0 && page < a.pages && key < k1;
        const long long at = page * a.page_stride + (key - split(key) * a.page) * a.kv_row;
        return {ok ? at : 0, __ballot(ok) | (KT == 64 ? 0 : ~0ull << 32)};
    }

    // ---- tiles: chunks of eight values, K's and then V's, dealt to the group's threads ----
    struct staged { raw r[NL]; };
    // x, new to the compiler here: what is made of it in a path seldom taken is made there, not kept in registers over the loop.
    static __device__ __forceinline__ int fresh(int x) {
        __asm__ volatile("" : "+v"(x));
        return x;
    }
    static __device__ __forceinline__ long long lane_of(long long v, int from) {
        return (long long)((unsigned long long)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), from) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, from));
    }
    // A load of the wave takes 64 / NC keys, which lie in one half of the tile.  Where a half cannot be on two pages, its place
    // is one number for the wave (a page's tokens past the last one are read, not used).
    __device__ __forceinline__ void fetch(staged& st, const spots& p) const {
        if (a.halves) {
            const uint32_t own = (lane / NC * (uint32_t)a.kv_row + 8 * (lane % NC)) * sizeof(KV);
            constexpr bool TWO = W == 16 && KT == 32;              // (kept where registers allow)
            long long half[2];
            if constexpr (TWO) {
                half[0] = lane_of(p.at, 0);
                half[1] = lane_of(p.at, 16);
            }
#pragma unroll
            for (int n = 0; n < NL; n++) {
                const int x0 = wr * 64 + n * GT, key0 = x0 / NC % KT;          // the wave's first
                const KV* const from = (x0 >= KT * NC ? V : K) + (TWO ? half[key0 / 16] : lane_of(p.at, key0 & ~15)) + (key0 & 15) * a.kv_row;
                st.r[n] = values_of::template load<WR == 1>((const KV*)((const char*)from + own));
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
            const int tg = fresh(this->tg);
#pragma unroll
            for (int n = 0; n < NL; n++) {
                const int x = tg + n * GT, key = x / NC % KT, c = x % NC;
                const long long at = __shfl(p.at, key) + 8 * c;
                st.r[n] = values_of::template load<WR == 1>((x >= KT * NC ? V : K) + at);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    // The addresses in one of the two buffers, new to the compiler in each round: kept over the loop, the sums made of them
    // would take half of the registers.
    struct addresses { uint32_t kr, vr, kw, vw; };
    __device__ __forceinline__ addresses tile_at(int buf) const {
        const uint32_t by = buf * REGION * 2;
        addresses t = {kr + by, vr + by, kw + by, vw + by};
        __asm__ volatile("" : "+v"(t.kr), "+v"(t.vr), "+v"(t.kw), "+v"(t.vw));
        return t;
    }
    template <typename T> static __device__ __forceinline__ auto lds_at(uint32_t p) { return (__attribute__((address_space(3))) T*)p; }
    __device__ __forceinline__ void stage(staged& st, unsigned long long valid, const addresses& t, keys& f) const {
        if (valid != ~0ull) {                         // keys that are not there become zeros
            const int tg = fresh(this->tg);
#pragma unroll
            for (int n = 0; n < NL; n++) {
                const int key = (tg + n * GT) / NC % KT;
                if (!(valid >> key & 1)) st.r[n] = raw{};
            }
        }
#pragma unroll
        for (int n = 0; n < NL; n++) {
            const int x = tg + n * GT, key = x / NC % KT, c = x % NC;
            constexpr int HALF = GT <= KT * NC ? NL / 2 : 0;       // of GT > KT NC threads half bring V
            const bool is_v = HALF ? n >= HALF : x >= KT * NC;
            const uint32_t p = is_v ? (t.vw ^ (W == 16 && GT / NC == 4 ? 32 * (n & 1) : 0)) + (n - HALF) * GT * 16 : (t.kw ^ 16 * (n * (GT / NC) / RPK % NC)) + n * GT * 16;
            if constexpr (NP == 1) {
                *lds_at<f16x8>(p) = st.r[n].a;
            } else {
                float y[8];
                float most = 0.0f;                    // (passes over NaN, which the products will show)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    y[e] = e < 4 ? st.r[n].a[e % 4] : st.r[n].b[e % 4];
                    most = fmaxf(most, fabsf(y[e]));
                }
                const uint32_t mx = lanes_max<NC>(__float_as_uint(most));
                const int ex = mx == 0 ? is_v ? kLeastV : 0 : row_scale(mx);   // (a row of zeros weighs nothing)
                const float up = pow2(-ex);
                f16x8 hi, lo;
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    f16x2 u, v;
                    split2(y[e] * up, y[e + 1] * up, u, v);
                    hi[e] = u[0];
                    hi[e + 1] = u[1];
                    lo[e] = v[0];
                    lo[e + 1] = v[1];
                }
                *lds_at<f16x8>(p) = hi;
                *lds_at<f16x8>(p + 2 * TILE) = lo;
                if (c == 0) {
                    if (is_v) {
                        f.v[key] = ex < kLeastV || ex > kMostV ? __builtin_nanf("") : (float)ex;
                        f.back[key] = up;
                    } else {
                        f.k[key] = pow2(ex - kLessK);
                    }
                }
            }
        }
    }

    // ---- products ----
    __device__ __forceinline__ void scores(acc (&s)[KB][SV], uint32_t kr) const {
#pragma unroll
        for (int i = 0; i < KB; i++)
#pragma unroll
            for (int n = 0; n < SQ; n++)
#pragma unroll
                for (int c = 0; c < 4; c++) set(s[i], n, c, 0.0f);
        f16x8 f[2][KB][SV][NP];                       // read one column of K ahead
        auto read = [&](int k) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < KB; i++)
#pragma unroll
                for (int j = 0; j < SV; j++)
#pragma unroll
                    for (int p = 0; p < NP; p++)
                        f[k & 1][i][j][p] = *lds_at<const f16x8>((kr ^ 16 * LR * k) + 2 * (p * TILE + (32 * i + 16 * j) * HD));
        };
        read(0);
#pragma unroll
        for (int k = 0; k < NK; k++) {
            if (k + 1 < NK) read(k + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < KB; i++)
#pragma unroll
                for (int j = 0; j < SV; j++)
#pragma unroll
                    for (int p = 2 - NP; p < 3; p++)  // the pieces' products, small ones first
                        s[i][j] = product(f[k & 1][i][j][p == 0 ? NP - 1 : 0], q[p == 1][k], s[i][j]);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    // V^T of W dims and 16 (W = 16: 32) keys from 16 g on: lane (dim lw, h) gets keys 4 h .. and 4 LR + 4 h ..
    __device__ __forceinline__ f16x8 transposed(uint32_t vr, int p, int j, int g) const {
        f16x8 r;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const s16x4 w = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)((vr ^ 2 * W * j) + 2 * (p * TILE + (16 * g + 4 * LR * e) * HD)));
            const f16x4 x = __builtin_bit_cast(f16x4, w);
#pragma unroll
            for (int k = 0; k < 4; k++) r[4 * e + k] = x[k];
        }
        return r;
    }
    // A factor of scores: not 0, as it multiplies masked ones (2^-149 at least; see kLessK.  Where the scale is 0, q is).
    static __device__ __forceinline__ float bounded(float x) { return fmaxf(x, 1.401298464e-45f); }
    __device__ __forceinline__ float factor_of_q() const { return __builtin_amdgcn_ldexpf(a.scale, NP == 2 ? qx + kLessK : qx) * kLog2e; }
    // A tile (KB of 32 keys): scores, the running maximum, weights, O.
    __device__ __forceinline__ void take(const addresses& t, const keys& f, int key, unsigned long long valid) {
        acc s[KB][SV];
        scores(s, t.kr);
        if (valid != ~0ull || have - key < KT) {
#pragma unroll
            for (int i = 0; i < KB; i++) {
                const uint32_t bits = (seen(key + 32 * i) & (uint32_t)(valid >> 32 * i)) >> (4 * h);
#pragma unroll
                for (int n = 0; n < SQ; n++)
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        if (!(bits >> (4 * LR * n + c) & 1)) set(s[i], n, c, -INFINITY);
            }
        }
        // The score in powers of two and V's scale, x + e, is s * factor + e0.  Mostly all keys of a tile have the same
        // scales, which WR = 4, bound by its vector instructions, makes use of (47.3 us without it, 44.9 with, in the case
        // above; one wave to a tile waits for memory, and gained nothing); else s becomes x + e itself.
        auto of = [&](const float (&x)[KT], int i, int n) __attribute__((always_inline)) {
            return *reinterpret_cast<const sgpu_f32x4*>(&x[32 * i + 4 * LR * n + 4 * h]);
        };
        float factor = bounded(factor_of_q()), e0 = 0.0f;
        bool same = NP == 1;
        if constexpr (NP == 2 && WR == 4) {
            const float k = f.k[lane % KT], e = f.v[lane % KT];
            const float k0 = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(k)));
            e0 = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(e)));
            same = __all(k == k0 && e == e0 && factor * k < INFINITY);
            if (same) factor = bounded(factor * k0);
        }
        if (!same) {
#pragma unroll
            for (int i = 0; i < KB; i++)
#pragma unroll
                for (int n = 0; n < SQ; n++) {
                    const sgpu_f32x4 kq = of(f.k, i, n), eq = of(f.v, i, n);
#pragma unroll
                    for (int c = 0; c < 4; c++) set(s[i], n, c, __builtin_fmaf(get(s[i], n, c) * kq[c], factor, eq[c]));
                }
            factor = 1.0f;
            e0 = 0.0f;
        }
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < KB; i++)
#pragma unroll
            for (int n = 0; n < SQ; n++)
#pragma unroll
                for (int c = 0; c < 4; c++) top = fmaxf(top, get(s[i], n, c));
        top = row_max(__builtin_fmaf(top, factor, e0));
        if (__any(top > m + LAG)) {                   // mostly at the first keys only
            const float mn = fmaxf(m, top), al = __builtin_amdgcn_exp2f(m - mn);
            l *= al;
#pragma unroll
            for (int n = 0; n < OQ; n++)
#pragma unroll
                for (int c = 0; c < 4; c++) set(o, n, c, get(o, n, c) * al);
            m = mn;
        }
        const float off = e0 + (OFF - m);
        constexpr int G = SQ / 2;                     // steps of the second product over 32 keys
        f16x8 ph[KB * G], pl[KB * G];
        float sum = 0.0f;
        if (!same) {
#pragma unroll
            for (int i = 0; i < KB; i++)
#pragma unroll
                for (int n = 0; n < SQ; n++) {
                    const sgpu_f32x4 back = of(f.back, i, n);
#pragma unroll
                    for (int c = 0; c < 4; c++) sum = __builtin_fmaf(__builtin_amdgcn_exp2f(get(s[i], n, c) + off), back[c], sum);
                }
            l += sum;
            sum = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < KB; i++)
#pragma unroll
            for (int n = 0; n < SQ; n++)
#pragma unroll
                for (int c = 0; c < 4; c += 2) {
                    float p[2];
                    f16x2 hi, lo;
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(get(s[i], n, c + j), factor, off));
                        sum += p[j];
                    }
                    split2(p[0], p[1], hi, lo);
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        ph[i * G + n / 2][n % 2 * 4 + c + j] = hi[j];
                        pl[i * G + n / 2][n % 2 * 4 + c + j] = lo[j];
                    }
                }
        if (same) l = NP == 2 ? __builtin_fmaf(sum, __builtin_amdgcn_exp2f(-e0), l) : l + sum;
        f16x8 v[2][NP];
        auto read = [&](int i) __attribute__((always_inline)) {
#pragma unroll
            for (int p = 0; p < NP; p++) v[i & 1][p] = transposed(t.vr, p, i % OV, i / OV * (2 / G));
        };
        read(0);
#pragma unroll
        for (int i = 0; i < KB * G * OV; i++) {
            const int j = i % OV, k = i / OV;
            if (i + 1 < KB * G * OV) read(i + 1);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (NP == 2) o[j] = product(v[i & 1][1], ph[k], o[j]);
            o[j] = product(v[i & 1][0], pl[k], o[j]);
            o[j] = product(v[i & 1][0], ph[k], o[j]);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    struct row_values { sgpu_f32x4 v[2 * NK]; };
    __device__ __forceinline__ void read_q(row_values& x) const {
#pragma unroll
        for (int k = 0; k < 2 * NK; k++) x.v[k] = *reinterpret_cast<const sgpu_f32x4*>(q_at + 8 * (LR * (k / 2) + h) + 4 * (k & 1));
    }
    __device__ __forceinline__ void cut_q(const row_values& x) {       // its scale joins the softmax's
        uint32_t mx = 0;
#pragma unroll
        for (int k = 0; k < 2 * NK; k++)
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const uint32_t u = __float_as_uint(x.v[k][c]) & 0x7fffffffu;
                mx = max(mx, u < 0x7f800000u ? u : 0u);
            }
        mx = max(mx, (uint32_t)__shfl_xor((int)mx, 32));
        if constexpr (LR == 4) mx = max(mx, (uint32_t)__shfl_xor((int)mx, 16));
        qx = scale_of(mx);
        // (a scale of 0: see bounded; one that leaves fp32 with q's: NaN, and so the vector ALUs' pass)
        const float up = !(a.scale > 0.0f) ? 0.0f : factor_of_q() < INFINITY ? pow2(-qx) : __builtin_nanf("");
#pragma unroll
        for (int k = 0; k < 2 * NK; k++)
#pragma unroll
            for (int c = 0; c < 4; c += 2) {
                f16x2 hi, lo;
                split2(x.v[k][c] * up, x.v[k][c + 1] * up, hi, lo);
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    q[0][k / 2][4 * (k & 1) + c + e] = hi[e];
                    q[1][k / 2][4 * (k & 1) + c + e] = lo[e];
                }
            }
    }
    __device__ __forceinline__ void clear(float m0) {
        m = m0;
        l = 0.0f;
#pragma unroll
        for (int n = 0; n < OQ; n++)
#pragma unroll
            for (int c = 0; c < 4; c++) set(o, n, c, 0.0f);
    }
    // Keys k0 .. k1-1: the key group's tiles k0 + 32 wk, a step of 32 WK from one to the next.  Ends with m, l the weights'
    // exponent and sum, o their average of V.
    __device__ __forceinline__ void run(int k0, int k1) {
        const int steps = (k1 - k0 + KT * WK - 1) / (KT * WK);
        int key = k0 + KT * wk;
        staged st;
        const int first = number(key);
        row_values x;
        read_q(x);
        __builtin_amdgcn_sched_barrier(0);
        spots p = find(key, first, k1);
        fetch(st, p);
        int next = number(key + KT * WK);
        __builtin_amdgcn_sched_barrier(0);
        cut_q(x);
        __builtin_amdgcn_sched_barrier(0);
        clear(-3e38f);                                // finite: what it is subtracted from may be -infinity
        for (int t = 0; t < steps; t++, key += KT * WK) {
            const addresses to = tile_at(t % BUFS);
            keys& f = info[NP == 2 ? t % BUFS : 0];
            const unsigned long long valid = p.valid;
            stage(st, valid, to, f);
            if (t + 1 < steps) {
                p = find(key + KT * WK, next, k1);
                fetch(st, p);
                next = number(key + 2 * KT * WK);
            }
            if constexpr (WR == 1) lds_sync();
            else __syncthreads();                     // the tile is in LDS, the other buffer free
            if (key < k1 && !idle) take(to, f, key, valid);
            if constexpr (WR == 1) lds_sync();
        }
        l = row_sum(l);
        float bad = l * 0.0f;
#pragma unroll
        for (int n = 0; n < OQ; n++)
#pragma unroll
            for (int c = 0; c < 4; c++) bad = __builtin_fmaf(get(o, n, c), 0.0f, bad);
        if (__any(live && bad != 0.0f)) {
            plain(k0 + KT * wk, k1);
            return;
        }
        const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
        for (int n = 0; n < OQ; n++)
#pragma unroll
            for (int c = 0; c < 4; c++) set(o, n, c, get(o, n, c) * inv);
        const int ex = l > 0.0f ? __builtin_amdgcn_frexp_expf(l) : 0;
        l = __builtin_amdgcn_ldexpf(l, -ex);
        m = l > 0.0f ? m - OFF + (float)ex : -INFINITY;
    }
    // The same, keys one after another, in fp32 on the vector ALUs, a lane's part of a score in 64 bits until it has its scale
    // (q.K alone may leave fp32's range).  (The barriers keep its registers few: they are the fast path's too.)
    __device__ __forceinline__ void plain(int first, int k1) {
        clear(-INFINITY);
        const int h = fresh(this->h);
        typedef KV quad __attribute__((ext_vector_type(4)));
#pragma unroll 1
        for (int n = 0, tile = first; tile < k1; n++, tile = first + n / KB * (KT * WK) + n % KB * 32) {
            const uint32_t bits = seen(tile);
#pragma unroll 1
            for (int u = 0; u < 32 && tile + u < k1; u++) {
                const bool mine = bits >> u & 1;
                if (!__any(mine)) continue;
                const int key = tile + u, page = page_of(a, b, key);
                if (page < 0) continue;
                const long long at = page * a.page_stride + key % a.page * a.kv_row;
                double part_of_x = 0.0;
#pragma unroll 1
                for (int d = 4 * h; d < HD; d += 4 * LR) {
                    const quad y = *reinterpret_cast<const quad*>(K + at + d);
                    const sgpu_f32x4 z = *reinterpret_cast<const sgpu_f32x4*>(q_at + d);
#pragma unroll
                    for (int e = 0; e < 4; e++) part_of_x = __builtin_fma((double)z[e], (double)y[e], part_of_x);
                }
                const double factor = 1.44269504088896340736 * (double)__int_as_float(fresh(__float_as_int(a.scale)));
                const float x = row_sum((float)(part_of_x * factor));
                if (!mine) continue;
                const float mn = fmaxf(m, x), base = mn == -INFINITY ? 0.0f : mn;
                const float al = __builtin_amdgcn_exp2f(m - base), p = __builtin_amdgcn_exp2f(x - base);
                const float ln = __builtin_fmaf(l, al, p), part = ln == 0.0f ? 0.0f : 1.0f / ln;
                const float keep = l * al * part, put = p * part;
                m = mn;
                l = ln;
#pragma unroll
                for (int n = 0; n < OQ; n++) {
                    const quad y = *reinterpret_cast<const quad*>(V + at + 4 * LR * n + 4 * h);
#pragma unroll
                    for (int c = 0; c < 4; c++) set(o, n, c, __builtin_fmaf(put, (float)y[c], get(o, n, c) * keep));
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
    }
    // The rows' averages to HD floats each (to: null where there is no row).
    __device__ __forceinline__ void put(float* to) const {
        if (to) {
#pragma unroll
            for (int n = 0; n < OQ; n++)
                *reinterpret_cast<sgpu_f32x4*>(to + 4 * LR * n + 4 * h) = sgpu_f32x4{get(o, n, 0), get(o, n, 1), get(o, n, 2), get(o, n, 3)};
        }
    }
};

// What bounds attention (us by the caller's clock, cold pages): few tokens, latency (one row of 700 tokens 10.4: lengths, table, page,
// join, each after the other); one or few rows a KV head, memory (64 requests of up to 4096 fp16 tokens, 82 MB, 22.5; two of
// 50001 with 7 rows each, 311 MB, 72, 4.3 TB/s); many rows, no one unit: 32 trees of 24 rows of up to 3001 fp32 tokens 39, in which
// a block takes 58k cycles, 29-31 at the 1.9-2.1 GHz that the card runs them at, and the last ends at 37-40; the vector ALUs
// (exponentials, the cutting of operands) issue for half of a wave's cycles, the matrix cores for a quarter, and waves wait for 37%.

// The batch as one line of steps: sequence by sequence its units (KV head, row tile), of each `start` steps for its beginning, then
// its steps of STEP keys (one where it has none).  Every wave works it out from the lengths on the device, 64 sequences at a time; the
// sums of up to 64 such runs tell where a step lies (each looked for from the first on, 512 sequences of 500 tokens took
// 44 us, so 36).
struct line_store { int q0[64], nq[64], have[64], N[64], tiles[64], steps[64], upto[64], sums[64], first, base, end; };
template <int ROWS, int STEP> struct tree_line {
    const tree_front& a;
    line_store& kept;                                 // of 64 sequences, from `first`, with steps base .. end-1: registers are the products'

    int total;                                        // all steps (the launcher's bound: below 2^30)
    struct sequence { int q0, nq, have, N, tiles, steps, upto; };      // rows, tokens in the cache, and with them; steps up to it and with it

    __device__ __forceinline__ tree_line(const tree_front& a_, line_store& k) : a(a_), kept(k) {}
    __device__ __forceinline__ sequence read(int b) const {
        sequence s;
        s.q0 = min(max(a.q_start[b], 0), a.R);
        s.nq = min(max(a.q_start[b + 1], 0), a.R) - s.q0;          // (below 0: starts that fall)
        s.have = min(max(a.len[b], 0), a.room);
        s.N = (int)min((long long)s.have + max(s.nq, 0), (long long)a.room);
        s.tiles = (s.nq * a.G + ROWS - 1) / ROWS;       // (R * NH is below 2^26)
        s.steps = max(1, (s.N + STEP - 1) / STEP);
        return s;
    }
    __device__ __forceinline__ sequence scan(int first) const {
        const int lane = threadIdx.x & 63, b = first + lane;
        sequence s = read(min(b, a.B - 1));
        s.upto = b < a.B ? a.NKV * s.tiles * (s.steps + a.start) : 0;
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            const int x = __shfl_up(s.upto, o);
            s.upto += lane >= o ? x : 0;
        }
        return s;
    }
    __device__ __forceinline__ void keep(const sequence& s) {      // (the waves write the same)
        const int lane = threadIdx.x & 63;
        kept.q0[lane] = s.q0;
        kept.nq[lane] = s.nq;
        kept.have[lane] = s.have;
        kept.N[lane] = s.N;
        kept.tiles[lane] = s.tiles;
        kept.steps[lane] = s.steps;
        kept.upto[lane] = s.upto;
        lds_sync();
    }
    __device__ __forceinline__ int runs() const { return (a.B + 4095) / 4096; }      // of 64 sequences, to one of the sums
    // (Starts that fall, which no batch has, could sum up to anything: nothing is done then.)
    __device__ __forceinline__ void measure() {
        bool falls = false;
        if (a.B <= 64) {
            const sequence s = scan(0);
            total = __builtin_amdgcn_readlane(s.upto, 63);
            falls = __any(s.nq < 0);
            keep(s);
        } else {
            const int lane = threadIdx.x & 63, per = runs(), last = (a.B - 1) / 64;
            total = 0;
            for (int n = 0; n <= last; n++) {
                const sequence s = scan(64 * n);
                total += __builtin_amdgcn_readlane(s.upto, 63);
                falls = falls || __any(s.nq < 0);
                if ((n + 1) % per == 0 || n == last) kept.sums[n / per] = total;
            }
            if (lane > last / per) kept.sums[lane] = total;
            kept.base = kept.end = 0;
            lds_sync();
        }
        if (falls) total = 0;
    }
    // The sequence with step x of the line, and its first step.  Called by all waves of a block with the same x.
    struct spot { int b, base; sequence s; };
    __device__ __forceinline__ spot find(int x) {
        int first = 0, base = 0;
        if (a.B > 64) {
            base = scalar(kept.base);
            if (x < base || x >= scalar(kept.end)) {
                __syncthreads();                      // no wave needs what is kept any more
                const int c = __builtin_ctzll(__ballot(kept.sums[threadIdx.x & 63] > x));
                int n = c * runs(), to;
                base = c ? scalar(kept.sums[c - 1]) : 0;
                for (;; n++, base = to) {
                    const sequence s = scan(64 * n);
                    to = base + __builtin_amdgcn_readlane(s.upto, 63);
                    if (x >= to) continue;
                    kept.first = 64 * n;
                    kept.base = base;
                    kept.end = to;
                    keep(s);
                    break;
                }
            }
            first = scalar(kept.first);
        }
        spot p;
        const int n = __builtin_ctzll(__ballot(kept.upto[threadIdx.x & 63] > x - base));
        p.b = first + n;
        p.s = {kept.q0[n], kept.nq[n], kept.have[n], kept.N[n], kept.tiles[n], kept.steps[n], base + kept.upto[n]};
        p.b = __builtin_amdgcn_readfirstlane(p.b);
        p.s = {scalar(p.s.q0), scalar(p.s.nq), scalar(p.s.have), scalar(p.s.N), scalar(p.s.tiles), scalar(p.s.steps), scalar(p.s.upto)};
        p.base = p.s.upto - a.NKV * p.s.tiles * (p.s.steps + a.start);
        return p;
    }
    static __device__ __forceinline__ int scalar(int v) { return __builtin_amdgcn_readfirstlane(v); }
};

// A block takes a run of the line's steps: the end of a unit, whole ones, the beginning of one.  What it has of a unit that
// is not whole goes to one of its two records: the second where the unit begins here, else the first.  Blocks are dealt
// to the 8 XCDs in turn: each XCD takes neighbouring runs, so that row tiles that read the same keys share an L2.
template <int HD, typename KV, int WR, int W>
__device__ __forceinline__ void tree(const tree_front& f, const paged_tree& a) {
    typedef tree_unit<HD, KV, WR, W> unit;
    constexpr int WK = unit::WK, ROWS = unit::ROWS, STEP = unit::KT * WK;
    __shared__ __attribute__((aligned(1024))) unsigned char lds[unit::BYTES];
    __shared__ __attribute__((aligned(16))) typename unit::keys info[unit::NP == 2 ? WK * unit::BUFS : 1];
    const int G = f.G;
    unit u(a, f, lds, info);
    // rows from v0 on against keys k0 .. k1-1; rec: the record's first row, or -1: the output's
    auto part_of = [&](int v0, int k0, int k1, int rec) __attribute__((always_inline)) {
        const int nv = u.nq * G;
        auto place = [&](int v) __attribute__((always_inline)) -> float* {
            const int i = f.row_of(v);
            return rec < 0 ? a.out + (u.q0 + i) * a.out_row + (u.g * G + v - i * G) * a.out_head : a.po + (size_t)(rec + v - v0) * HD;
        };
        auto record = [&](int v, float m, float l) __attribute__((always_inline)) {
            if (rec >= 0) *reinterpret_cast<f32x2*>(a.pml + 2 * (size_t)(rec + v - v0)) = f32x2{m, l};
        };
        u.rows(v0);
        u.run(k0, k1);
        if constexpr (WK == 1) {
            const int v = v0 + W * u.wr + unit::fresh(u.lw);
            u.put(u.live ? place(v) : nullptr);
            if (u.live && u.h == 0) record(v, u.m, u.l);
            __syncthreads();                          // the buffers are the next rows'
        } else {                                      // merge the key groups
            float (*part)[HD + 4] = reinterpret_cast<float (*)[HD + 4]>(lds), *const ml = reinterpret_cast<float*>(lds) + 4 * W * (HD + 4);
            __syncthreads();
            const int mine = W * u.wave + unit::fresh(u.lw);       // (key group, row) = wave / WR, W (wave % WR) + lw
            u.put(part[mine]);
            if (u.h == 0) {
                ml[mine] = u.m;
                ml[4 * W + mine] = u.l;
            }
            __syncthreads();
            constexpr int PER = 256 / ROWS, D = HD / PER;          // threads of a row, their dims
            const int tid = unit::fresh(threadIdx.x), w = tid / PER, d0 = tid % PER * D, v = v0 + w;
            if (v < nv) {
                float M = -INFINITY, L = 0.0f, x[D];
#pragma unroll
                for (int k = 0; k < WK; k++) M = fmaxf(M, ml[k * ROWS + w]);
                const float base = M == -INFINITY ? 0.0f : M;
#pragma unroll
                for (int e = 0; e < D; e++) x[e] = 0.0f;
#pragma unroll
                for (int k = 0; k < WK; k++) L += ml[4 * W + k * ROWS + w] * __builtin_amdgcn_exp2f(ml[k * ROWS + w] - base);
#pragma unroll
                for (int k = 0; k < WK; k++) {
                    const float lk = ml[4 * W + k * ROWS + w];
                    if (lk == 0.0f) continue;         // this group saw nothing of the row
                    const float wt = lk * __builtin_amdgcn_exp2f(ml[k * ROWS + w] - base) / L;
#pragma unroll
                    for (int e = 0; e < D; e++) x[e] = __builtin_fmaf(part[k * ROWS + w][d0 + e], wt, x[e]);
                }
                if (d0 == 0) record(v, M, L);
                float* const to = place(v) + d0;
#pragma unroll
                for (int e = 0; e < D; e += D < 4 ? 2 : 4) {
                    if constexpr (D < 4) *reinterpret_cast<f32x2*>(to + e) = f32x2{x[e], x[e + 1]};
                    else *reinterpret_cast<sgpu_f32x4*>(to + e) = sgpu_f32x4{x[e], x[e + 1], x[e + 2], x[e + 3]};
                }
            }
            __syncthreads();
        }
    };
    const bool dealt = f.NB > 0;
    int x, end, run = 0, block = 0;                   // the steps of this block (dealt), or its first row of a tile
    __shared__ line_store kept;
    tree_line<ROWS, STEP> line(f, kept);
    if (dealt) {
        // rows of no sequence: nothing to join
        for (int i = blockIdx.x * 256 + threadIdx.x, q0 = min(max(f.q_start[0], 0), f.R), q1 = min(max(f.q_start[f.B], q0), f.R);
             i < (q0 + f.R - q1) * a.NH; i += f.NB * 256)
            a.desc[2 * ((long long)i + (i < q0 * a.NH ? 0 : (q1 - q0) * a.NH)) + 1] = 0;
        line.measure();
        if (line.total == 0)
            for (int i = blockIdx.x * 256 + threadIdx.x; i < f.R * a.NH; i += f.NB * 256) a.desc[2 * (long long)i + 1] = 0;
        run = (line.total + f.NB - 1) / f.NB;
        const int xcd = blockIdx.x % 8;
        block = xcd * (f.NB / 8) + min(xcd, f.NB % 8) + blockIdx.x / 8;
        x = (int)min((long long)block * run, (long long)line.total);
        end = (int)min((long long)x + run, (long long)line.total);
    } else {
        const int rest = blockIdx.x / (8 * a.MT) * 8 + blockIdx.x % 8;
        if (rest >= f.B * f.NKV) return;
        const auto q = line.read(rest / f.NKV);
        u.sequence(rest / f.NKV, rest % f.NKV, q.q0, q.nq, q.have, q.N);
        x = blockIdx.x / 8 % a.MT * ROWS;
        end = u.nq * G;
    }
    while (x < end) {
        int v0 = x, k0 = 0, k1 = u.N, rec = -1, next = x + a.MT * ROWS, last = 0;
        bool tell = false;
        if (dealt) {
            const auto at = line.find(x);
            const int steps = at.s.steps, S = steps + f.start;
            const int n = (x - at.base) / S, y = x - at.base - n * S, count = min(S - y, end - x);
            next = x + count;
            const int t = max(y - f.start, 0), stop = y + count - f.start;          // the unit's own steps t .. stop-1
            if (stop <= t) {
                x = next;
                continue;
            }
            u.sequence(at.b, n / at.s.tiles, at.s.q0, at.s.nq, at.s.have, at.s.N);
            v0 = n % at.s.tiles * ROWS;
            k0 = min(t * STEP, u.N);
            k1 = (int)min((long long)stop * STEP, (long long)u.N);
            if (stop - t < steps) rec = (2 * block + (t == 0)) * ROWS;
            tell = t == 0;
            last = x - y + S - 1;
        }
        part_of(v0, k0, k1, rec);
        if (tell) {                                   // where the unit begins: for the join
            const int w = unit::fresh(threadIdx.x), v = v0 + w;
            if (w < ROWS && v < u.nq * G) {
                const int i = f.row_of(v);
                *reinterpret_cast<i32x2*>(a.desc + 2 * ((long long)(u.q0 + i) * a.NH + u.g * G + v - i * G)) =
                    i32x2{block << 8 | w, rec < 0 ? 0 : last / run - block + 1};
            }
        }
        x = next;
    }
}

// The records of each row and head joined, a wave each: 64 / T records side by side, HD = 4 T dims, eight of each on their way
// at once.
template <int HD>
__device__ __forceinline__ void tree_join(const int* __restrict__ desc, const float* __restrict__ po, const float* __restrict__ pml, float* __restrict__ out,
                                          long long out_row, long long out_head, int NH, int n, int rows) {
    constexpr int T = HD / 4, P = 64 / T, U = 8;
    const int t = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (t >= n) return;
    const i32x2 told = *reinterpret_cast<const i32x2*>(desc + 2 * (long long)t);
    const int where = told[0], S = told[1], lane = threadIdx.x & 63, part = lane / T, d = lane % T * 4;
    if (S == 0) return;
    const int r = t / NH, hd = t - r * NH;
    const int block = where >> 8, w0 = where & 255;
    auto rec = [&](int s) __attribute__((always_inline)) { return (size_t)(2 * (block + s) + (s == 0)) * rows + w0; };
    float M = -INFINITY, L = 0.0f;
    sgpu_f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s0 = 0; s0 < S; s0 += 64) {
        f32x2 y = {-INFINITY, 0.0f};
        if (s0 + lane < S) y = *reinterpret_cast<const f32x2*>(pml + 2 * rec(s0 + lane));
        float w = 0.0f;
        for (int k0 = 0; k0 < 64 && s0 + k0 < S; k0 += U * P) {
            sgpu_f32x4 v[U];
#pragma unroll
            for (int k = 0; k < U; k++) v[k] = *reinterpret_cast<const sgpu_f32x4*>(po + rec(min(s0 + k0 + k * P + part, S - 1)) * HD + d);
            if (k0 == 0) {
                if (y[1] == 0.0f) y = f32x2{-INFINITY, 0.0f};      // nothing seen
                const float mn = fmaxf(M, sgpu_wave_max(y[0])), base = mn == -INFINITY ? 0.0f : mn;
                const float al = __builtin_amdgcn_exp2f(M - base);
                M = mn;
                w = y[1] == 0.0f ? 0.0f : y[1] * __builtin_amdgcn_exp2f(y[0] - base);
                L = __builtin_fmaf(L, al, sgpu_wave_sum(w));
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] *= al;
            }
#pragma unroll
            for (int k = 0; k < U; k++) {
                const int s = k0 + k * P + part;
                const float ws = __shfl(w, s & 63);
                if (s < 64 && ws != 0.0f) {           // (a NaN is not 0)
#pragma unroll
                    for (int e = 0; e < 4; e++) x[e] = __builtin_fmaf(v[k][e], ws, x[e]);
                }
            }
        }
    }
#pragma unroll
    for (int o = T; o < 64; o *= 2)
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] += __shfl_xor(x[e], o);
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] = L == 0.0f ? 0.0f : x[e] / L;
    if (part == 0) *reinterpret_cast<sgpu_f32x4*>(out + r * out_row + hd * out_head + d) = x;
}

// ---- logits ----
constexpr int kLogits = 8192;             // values of a chunk: eight a thread
constexpr int kTokens = 4;                // tokens of the history that a thread keeps

// A run of row r's chunks.  For each, the row's tokens that fall into it are counted in LDS (whole numbers: their order
// does not matter), the latest of a token's biases found, and then each value is read, adjusted and written once, the
// next chunk's on their way.  The first 4096 tokens and 1024 biases of the row stay in registers from chunk to chunk.  What
// a penalty or bias touches is computed in 64 bits and rounded once.  In place, only what changes is read or written.
// Bound by memory: 512 fp16 rows of 151936 under a grammar that allows 2% (328 MB counted whole) 67 us, 4.9 TB/s; 68 rows of 50257,
// half allowed, 9.0 (3.1 TB/s: one chunk a block, its tables before its values); one row 4.7, latency.  Two blocks a CU: 512
// of 1024 threads in all (68 rows 10.9 us with 256, 9.5 with 512 or 1024; 100 rows of 151936 26.7, 18.5, 20.0).
template <typename X, bool BIAS>
__device__ __forceinline__ void logits(const paged_logits& a) {
    __shared__ __attribute__((aligned(16))) uint32_t said[kLogits], last[BIAS ? kLogits : 4];
    __shared__ float biases[BIAS ? 1024 : 1];
    __shared__ uint32_t map[kLogits / 32];            // of the values that have an entry in the tables: the rest of those is not read
    typedef X vec __attribute__((ext_vector_type(8), aligned(sizeof(X))));
    const int tid = threadIdx.x, r = blockIdx.x / a.groups, e0 = 8 * tid, per = (a.C + a.groups - 1) / a.groups;
    const int c0 = blockIdx.x % a.groups * per, c1 = min(c0 + per, a.C);
    const X* const x = (const X*)a.x + r * a.x_row + e0;
    X* const y = (X*)a.y + r * a.y_row + e0;
    const uint8_t* const allowed = a.allow ? (const uint8_t*)(a.allow + r * a.allow_row) + tid : nullptr;
    const bool same = a.x == a.y;
    // the eight values' bits of the grammar (0 past the row: nothing to do), the values themselves where any is allowed
    auto bits_of = [&](int c) __attribute__((always_inline)) -> uint32_t {
        const int v = c * kLogits + e0;
        return c >= c1 || v >= a.V ? 0 : allowed ? allowed[c * (kLogits / 8)] : 0xff;
    };
    auto values_of = [&](int c, uint32_t bits) __attribute__((always_inline)) -> vec {
        vec v = {};
        const int at = c * kLogits;
        if (bits != 0 && at + e0 + 8 <= a.V) {
            v = *reinterpret_cast<const vec*>(x + at);
        } else if (bits != 0) {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (at + e0 + j < a.V) v[j] = x[at + j];
        }
        return v;
    };
    uint32_t bits = bits_of(c0), next_bits = bits_of(c0 + 1);
    vec in = {};
    if (!same) in = values_of(c0, bits);
    const sgpu_u32x4 none = {0, 0, 0, 0};
    if (tid < kLogits / 32) map[tid] = 0;
    for (int j = 0; j < 8; j += 4) {
        *reinterpret_cast<sgpu_u32x4*>(said + e0 + j) = none;
        if constexpr (BIAS) *reinterpret_cast<sgpu_u32x4*>(last + e0 + j) = none;
    }
    // the row's tokens: its prompt's, then its output's
    uint32_t from[2] = {0, 0}, n[2] = {0, 0};
    if (a.span) {
#pragma unroll
        for (int k = 0; k < 2; k++) {
            from[k] = min(max(a.span[4ll * r + 2 * k], 0), a.n_tok);
            n[k] = min(max(a.span[4ll * r + 2 * k + 1], 0), a.n_tok - (int)from[k]);
        }
    }
    const uint32_t all = n[0] + n[1];                 // (each below 2^31)
    auto token = [&](uint32_t j) __attribute__((always_inline)) { return j >= all ? -1 : a.tok[j < n[0] ? from[0] + j : from[1] - n[0] + j]; };
    int kept[kTokens];
#pragma unroll
    for (int i = 0; i < kTokens; i++) kept[i] = token(tid + 1024 * i);
    int b0 = 0, nb = 0, kept_id = -1;
    if constexpr (BIAS) {
        b0 = min(max(a.bias_span[2ll * r], 0), a.n_bias);
        nb = min(max(a.bias_span[2ll * r + 1], 0), a.n_bias - b0);
        if (tid < nb) {
            kept_id = a.bias_id[b0 + tid];
            biases[tid] = a.bias[b0 + tid];
        }
    }
    const double more = a.rep ? a.rep[r] : 1.0f, less = 1.0 / more;
    const float freq = a.freq ? a.freq[r] : 0.0f, pres = a.pres ? a.pres[r] : 0.0f;
    __syncthreads();
    for (int c = c0; c < c1; c++) {
        const int v0 = c * kLogits, left = a.V - v0;               // (left: at least one)
        const uint32_t size = (uint32_t)min(left, kLogits);
        auto count = [&](int id, bool output) __attribute__((always_inline)) {     // prompt: bit 31; output: counted
            const uint32_t at = (uint32_t)id - (uint32_t)v0;
            if (id < 0 || at >= size) return;
            atomicOr(&map[at / 32], 1u << at % 32);
            if (output) atomicAdd(&said[at], 1u);
            else atomicOr(&said[at], 0x80000000u);
        };
#pragma unroll
        for (int i = 0; i < kTokens; i++) count(kept[i], tid + 1024 * i >= n[0]);
        for (uint32_t j = tid + 1024 * kTokens; j < all && j >= 1024; j += 1024) count(token(j), j >= n[0]);
        if constexpr (BIAS) {
            auto bias = [&](int id, int j) __attribute__((always_inline)) {
                const uint32_t at = (uint32_t)id - (uint32_t)v0;
                if (id < 0 || at >= size) return;
                atomicOr(&map[at / 32], 1u << at % 32);
                atomicMax(&last[at], (uint32_t)j + 1u);
            };
            bias(kept_id, tid);
            for (int j = tid + 1024; j < nb; j += 1024) bias(a.bias_id[b0 + j], j);
        }
        const vec after = same ? vec{} : values_of(c + 1, next_bits);
        const uint32_t after_bits = bits_of(c + 2);
        __syncthreads();
        const uint32_t touched = reinterpret_cast<const uint8_t*>(map)[tid];       // of the eight values
        if (e0 < left && !(same && touched == 0 && bits == 0xff)) {
            if (same && bits != 0) in = values_of(c, bits);
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (!(bits >> j & 1)) in[j] = (X)-INFINITY;
            if (left - e0 >= 8) {
                *reinterpret_cast<vec*>(y + v0) = in;
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (e0 + j < left) y[v0 + j] = in[j];
            }
            // the few that a penalty or bias touches, one by one (all eight at once take twice the registers)
            for (uint32_t t = touched & bits; t; t &= t - 1) {
                const int j = __builtin_ctz(t);
                const uint32_t w = said[e0 + j], times = w & 0x7fffffffu;
                X from_row = in[0];
#pragma unroll
                for (int k = 1; k < 8; k++) from_row = j == k ? in[k] : from_row;
                double z = (double)from_row;
                if (w) z *= z > 0.0 ? less : more;
                if (times) z = z - (double)freq * (double)times - (double)pres;
                if constexpr (BIAS) {
                    const int i = (int)last[e0 + j] - 1;
                    if (i >= 0) z += (double)(i < 1024 ? biases[i] : a.bias[b0 + i]);
                }
                y[v0 + j] = (X)z;
            }
        }
        if (touched) {                                // for the next chunk
            reinterpret_cast<uint8_t*>(map)[tid] = 0;
            for (int j = 0; j < 8; j += 4) {
                *reinterpret_cast<sgpu_u32x4*>(said + e0 + j) = none;
                if constexpr (BIAS) *reinterpret_cast<sgpu_u32x4*>(last + e0 + j) = none;
            }
        }
        in = after;
        bits = next_bits;
        next_bits = after_bits;
        __syncthreads();
    }
}

}  // namespace

#define SGPU_HEADS(NAME, QO, KO, PAGED, VEC, ONCE)                                                                    \
    extern "C" __global__ void __launch_bounds__(256) sgpu_heads_##NAME(paged_heads a) { heads<QO, KO, PAGED, VEC, ONCE>(a); }
SGPU_HEADS(rows_f32, float, float, false, false, false)
SGPU_HEADS(rows_f16, _Float16, _Float16, false, false, false)
SGPU_HEADS(rows_v8_f32, float, float, false, true, false)
SGPU_HEADS(rows_v8_f16, _Float16, _Float16, false, true, false)
SGPU_HEADS(rows_v8s_f32, float, float, false, true, true)
SGPU_HEADS(rows_v8s_f16, _Float16, _Float16, false, true, true)
SGPU_HEADS(pages_f32, float, float, true, false, false)
SGPU_HEADS(pages_f16, float, _Float16, true, false, false)
SGPU_HEADS(pages_v8_f32, float, float, true, true, false)
SGPU_HEADS(pages_v8_f16, float, _Float16, true, true, false)
SGPU_HEADS(pages_v8s_f32, float, float, true, true, true)
SGPU_HEADS(pages_v8s_f16, float, _Float16, true, true, true)

#define SGPU_TREE_KERNEL(HD, KV, NAME, WR, W, WAVES)                                                                  \
    extern "C" __global__ void __launch_bounds__(256, WAVES) sgpu_tree_##NAME##_##HD(                                 \
        const int* q_start, const int* len, int B, int R, int NKV, int G, int room, int NB, int start, int magic, paged_tree a) { \
        const tree_front f = {q_start, len, B, R, NKV, G, room, NB, start, magic};                                    \
        tree<HD, KV, WR, W>(f, a);                                                                                    \
    }
#define SGPU_TREE(HD)                                                                                                 \
    SGPU_TREE_KERNEL(HD, float, r16_f32, 1, 16, (HD) <= 64 ? 2 : 1)                                                   \
    SGPU_TREE_KERNEL(HD, float, r32_f32, 1, 32, (HD) <= 64 ? 2 : 1)                                                   \
    SGPU_TREE_KERNEL(HD, float, r64_f32, 2, 32, (HD) <= 64 ? 2 : 1)                                                   \
    SGPU_TREE_KERNEL(HD, float, r128_f32, 4, 32, 2)                                                                   \
    SGPU_TREE_KERNEL(HD, _Float16, r16_f16, 1, 16, (HD) <= 64 ? 4 : 2)                                                \
    SGPU_TREE_KERNEL(HD, _Float16, r32_f16, 1, 32, 2)                                                                 \
    SGPU_TREE_KERNEL(HD, _Float16, r64_f16, 2, 32, 2)                                                                 \
    SGPU_TREE_KERNEL(HD, _Float16, r128_f16, 4, 32, 2)                                                                \
    extern "C" __global__ void __launch_bounds__(256) sgpu_tree_join_##HD(                                            \
        const int* __restrict__ desc, const float* __restrict__ po, const float* __restrict__ pml, float* __restrict__ out, \
        long long out_row, long long out_head, int NH, int n, int rows) {                                             \
        tree_join<HD>(desc, po, pml, out, out_row, out_head, NH, n, rows);                                            \
    }
SGPU_TREE(32)
SGPU_TREE(64)
SGPU_TREE(128)

#define SGPU_LOGITS(NAME, X, BIAS)                                                                                    \
    extern "C" __global__ void __launch_bounds__(1024, 8) sgpu_logits_##NAME(paged_logits a) { logits<X, BIAS>(a); }
SGPU_LOGITS(f32, float, false)
SGPU_LOGITS(f16, _Float16, false)
SGPU_LOGITS(bias_f32, float, true)
SGPU_LOGITS(bias_f16, _Float16, true)
