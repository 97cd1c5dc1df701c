// sgpu_paged.hip -- what a host that serves several requests from one paged cache, and checks tokens drafted
// ahead, needs beside the decode engines' own kernels (gfx950):
//   sgpu_heads_*    each head's norm and rotation, into rows or into the pages of a cache
//   sgpu_tree_*     attention of new rows over their sequence's pages, with a tree's mask over the new ones
//   sgpu_logits_*   penalties, biases and a grammar's mask on logits
// fp16 values here are IEEE ones, as in sgpu_score.hip.
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
    int T, NH, NKV, HD, tb, team;         // rows a block, log2 of a head's lanes
    int pages, page, table_pages, B;
};
struct paged_tree {
    const void *k, *v;
    const float* q;
    float* out;
    const int *table, *len, *q_start;
    const uint32_t* mask;
    float *po, *pml;                      // partial outputs, and (max, sum, splits, -) of each: [split][row][head]
    long long page_stride, kv_row, kv_head, table_row, q_row, q_head, out_row, out_head, mask_row;
    int pages, page, table_pages, R, B, NH, NKV;
    float scale;
    int S, chunk, MT;                     // splits of the keys, keys of one, row tiles
};
struct paged_logits {
    const void* x;
    void* y;
    const int *tok, *span, *bias_id, *bias_span;
    const float *rep, *freq, *pres, *bias;
    const uint32_t* allow;
    long long x_row, y_row, allow_row;
    int rows, V, n_tok, n_bias, C;        // C: chunks of a row
};

namespace {

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

// 1 / sqrt(x): the 64-bit approximation and one step of Newton's method (2^-46 or better).
__device__ __forceinline__ double inv_sqrt(double x) {
    const double y = __builtin_amdgcn_rsq(x);
    return y * (1.5 - 0.5 * x * y * y);
}
__device__ __forceinline__ double lanes_sum(double s, int lanes) {
    for (int o = 1; o < lanes; o *= 2) s += __shfl_xor(s, o);
    return s;
}

// Rows t of q (NH heads), k (NKV) and, into pages, v (NKV): y = rot(x * w / sqrt(mean x^2 + eps)), the norm where
// there are weights, its squares summed in 64 bits (no value's square leaves them); v as it is.  Pair i of a head is (i, i + rot/2),
// or (2i, 2i+1), and turns by turns[i] per position.  PAGED: row t is token len[b] + i of its sequence b, k and v go to
// its place in the pages (rows without one are left out), and rows of no sequence are left as they were.
// A block takes tb rows: their places and angles once into LDS, then every head reads them.  VEC: 2^team lanes a
// head, eight values each (a pair's both sides in one lane); otherwise a wave a head, a pair or a value a lane.
// In place is fine: a head's values are all read before the first is written.
template <typename QO, typename KO, bool PAGED, bool VEC>
__device__ __forceinline__ void heads(const paged_heads& a) {
    __shared__ float table[2 * kAngles];
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
                const bool live = e < HD / 8, turn = e < rot / 8;
                const bool apart = turn && !a.neighbours;
                const int d0 = apart ? 4 * e : 8 * e, d1 = apart ? half + 4 * e : 8 * e + 4;
                float u[4] = {}, v[4] = {};
                if (live) {
                    const sgpu_f32x4 p = *reinterpret_cast<const sgpu_f32x4*>(x + d0), q = *reinterpret_cast<const sgpu_f32x4*>(x + d1);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        u[j] = p[j];
                        v[j] = q[j];
                    }
                }
                if (w) {
                    double s = 0.0;
#pragma unroll
                    for (int j = 0; j < 4; j++) s += (double)u[j] * u[j] + (double)v[j] * v[j];
                    const float r = (float)inv_sqrt(lanes_sum(s, lanes) / HD + a.eps);
                    if (live) {
                        const sgpu_f32x4 p = *reinterpret_cast<const sgpu_f32x4*>(w + d0), q = *reinterpret_cast<const sgpu_f32x4*>(w + d1);
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            u[j] = u[j] * r * p[j];
                            v[j] = v[j] * r * q[j];
                        }
                    }
                }
                if (!live) continue;
                if (apart) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float c = tab[2 * (4 * e + j)], s = tab[2 * (4 * e + j) + 1], p = u[j];
                        u[j] = p * c - v[j] * s;
                        v[j] = p * s + v[j] * c;
                    }
                } else if (turn) {
                    const float* const k = tab + 8 * e;
                    const float p[8] = {u[0] * k[0] - u[1] * k[1], u[0] * k[1] + u[1] * k[0], u[2] * k[2] - u[3] * k[3],
                                        u[2] * k[3] + u[3] * k[2], v[0] * k[4] - v[1] * k[5], v[0] * k[5] + v[1] * k[4],
                                        v[2] * k[6] - v[3] * k[7], v[2] * k[7] + v[3] * k[6]};
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        u[j] = p[j];
                        v[j] = p[4 + j];
                    }
                }
                if (kind == 0) {
                    put4(yq + d0, u);
                    put4(yq + d1, v);
                } else {
                    put4(yk + d0, u);
                    put4(yk + d1, v);
                }
            } else {
                float r = 1.0f;
                if (w) {
                    double s = 0.0;
                    for (int d = e; d < HD; d += 64) s += (double)x[d] * x[d];
                    r = (float)inv_sqrt(lanes_sum(s, 64) / HD + a.eps);
                }
                auto at = [&](int d) __attribute__((always_inline)) { return w ? x[d] * r * w[d] : x[d]; };
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
template <int HD, typename KV> struct tree_unit {
    static constexpr int ND = HD / 32, ROWS = 32;

    const paged_tree& a;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l32 = lane & 31, h = lane >> 5;
    int b, g, q0, nq, have, N, i;                     // the sequence, KV head, its rows and keys; this lane's row of it
    bool live;                                        // there is such a row
    const float* q_at;
    float m, l, o[ND][16];                            // max and sum of the weights, their average of V: dim 32j + 8(e/4) + 4h + e%4

    __device__ __forceinline__ tree_unit(const paged_tree& a_) : a(a_) {}
    __device__ __forceinline__ void sequence(int b_, int g_) {
        b = b_;
        g = g_;
        q0 = min(max(a.q_start[b], 0), a.R);
        nq = min(max(a.q_start[b + 1], q0), a.R) - q0;
        const int room = a.table_pages * a.page;
        have = min(max(a.len[b], 0), room);
        N = min(have + nq, room);                     // (both below 2^30)
    }
    __device__ __forceinline__ void rows(int v) {     // v: row and head of the group, G = NH / NKV to a row
        const int G = a.NH / a.NKV, nv = nq * G, w = min(v, nv - 1);
        live = v < nv;
        i = w / G;
        q_at = a.q + (q0 + i) * a.q_row + (g * G + w - i * G) * a.q_head;
    }
    // Which of the 32 keys from `key` on this lane's row sees, a bit each.
    __device__ __forceinline__ uint32_t seen(int key) const {
        if (!live) return 0;
        const int old = have - key, j = key - have;
        if (old >= 32) return ~0u;
        uint32_t bits;
        if (!a.mask) {
            const int c = i - j + 1;                  // the keys up to the row's own
            bits = c >= 32 ? ~0u : c > 0 ? (1u << c) - 1 : 0;
        } else {
            const uint32_t* const w = a.mask + (q0 + i) * a.mask_row;
            if (old > 0) {
                bits = (a.mask_row > 0 ? w[0] << old : 0) | ((1u << old) - 1);
            } else {
                const int at = j / 32, s = j % 32;
                bits = at < a.mask_row ? w[at] >> s : 0;
                if (s && at + 1 < a.mask_row) bits |= w[at + 1] << (32 - s);
            }
        }
        const int left = N - key;
        return left >= 32 ? bits : left > 0 ? bits & ((1u << left) - 1) : 0;
    }

    __device__ __forceinline__ void clear() {
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int j = 0; j < ND; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) o[j][e] = 0.0f;
    }
    // Keys k0 .. k1-1 (32 at a time, every STEP from `k0` on) one after another, in fp32 on the vector ALUs.
    __device__ void plain(int k0, int k1, int step) {
        clear();
        float q[ND][16];
#pragma unroll
        for (int j = 0; j < ND; j++)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const sgpu_f32x4 x = *reinterpret_cast<const sgpu_f32x4*>(q_at + 32 * j + 2 * e + 4 * h);
#pragma unroll
                for (int c = 0; c < 4; c++) q[j][e + c] = x[c] ;
            }
        typedef KV quad __attribute__((ext_vector_type(4)));
        for (int tile = k0; tile < k1; tile += step) {
            const uint32_t bits = seen(tile);
            for (int u = 0; u < 32 && tile + u < k1; u++) {
                const bool mine = bits >> u & 1;
                if (!__any(mine)) continue;
                const int key = tile + u, page = page_of(a, b, key);
                if (page < 0) continue;
                const long long at = page * a.page_stride + key % a.page * a.kv_row + g * a.kv_head;
                const KV *const kr = (const KV*)a.k + at, *const vr = (const KV*)a.v + at;
                float x = 0.0f;
#pragma unroll
                for (int j = 0; j < ND; j++)
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        const quad y = *reinterpret_cast<const quad*>(kr + 32 * j + 2 * e + 4 * h);
#pragma unroll
                        for (int c = 0; c < 4; c++) x = __builtin_fmaf(q[j][e + c], (float)y[c], x);
                    }
                x = half_sum(x) * (a.scale * kLog2e);
                if (!mine) continue;
                const float mn = fmaxf(m, x), base = mn == -INFINITY ? 0.0f : mn;
                const float al = __builtin_amdgcn_exp2f(m - base), p = __builtin_amdgcn_exp2f(x - base);
                const float ln = __builtin_fmaf(l, al, p), part = ln == 0.0f ? 0.0f : 1.0f / ln;
                const float keep = l * al * part, put = p * part;
                m = mn;
                l = ln;
#pragma unroll
                for (int j = 0; j < ND; j++)
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        const quad y = *reinterpret_cast<const quad*>(vr + 32 * j + 2 * e + 4 * h);
#pragma unroll
                        for (int c = 0; c < 4; c++) o[j][e + c] = __builtin_fmaf(put, (float)y[c], o[j][e + c] * keep);
                    }
            }
        }
    }
};

// The rows of one sequence and KV head (32 a tile, a lane pair each) over the keys of one split; the block's four
// waves take 32 keys in turn and are merged at the end.  Blocks of the row tiles that read the same keys share an XCD
// (blocks are dealt to the 8 XCDs in turn).
template <int HD, typename KV>
__device__ __forceinline__ void tree(const paged_tree& a) {
    constexpr int ND = HD / 32, ROWS = 32;
    __shared__ float part[4][32][HD + 1], ml[4][2][32];
    const int rest = blockIdx.x / (8 * a.MT) * 8 + blockIdx.x % 8, mt = blockIdx.x / 8 % a.MT;
    if (rest >= a.B * a.NKV * a.S) return;
    const int s = rest % a.S, g = rest / a.S % a.NKV, G = a.NH / a.NKV;
    tree_unit<HD, KV> u(a);
    u.sequence(rest / a.S / a.NKV, g);
    const int k0 = min((long long)s * a.chunk, (long long)u.N), k1 = s == a.S - 1 ? u.N : min((long long)k0 + a.chunk, (long long)u.N);
    const int used = min(a.S, max(1, (u.N + a.chunk - 1) / a.chunk));
    if (s >= used) return;
    for (int v0 = mt * ROWS; v0 < u.nq * G; v0 += a.MT * ROWS) {
        u.rows(v0 + u.l32);
        u.plain(k0 + 32 * u.wave, k1, 128);
#pragma unroll
        for (int j = 0; j < ND; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) part[u.wave][u.l32][32 * j + 8 * (e / 4) + 4 * u.h + e % 4] = u.o[j][e];
        if (u.h == 0) {
            ml[u.wave][0][u.l32] = u.m;
            ml[u.wave][1][u.l32] = u.l;
        }
        __syncthreads();
        // 8 threads a row, HD / 8 dims each
        const int w = threadIdx.x / 8, d0 = threadIdx.x % 8 * (HD / 8), v = v0 + w;
        if (v < u.nq * G) {
            float M = -INFINITY, L = 0.0f, x[HD / 8];
#pragma unroll
            for (int k = 0; k < 4; k++) M = fmaxf(M, ml[k][0][w]);
            const float base = M == -INFINITY ? 0.0f : M;
#pragma unroll
            for (int e = 0; e < HD / 8; e++) x[e] = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; k++) L += ml[k][1][w] * __builtin_amdgcn_exp2f(ml[k][0][w] - base);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (ml[k][1][w] == 0.0f) continue;     // this wave saw nothing of the row
                const float wt = ml[k][1][w] * __builtin_amdgcn_exp2f(ml[k][0][w] - base) / L;
#pragma unroll
                for (int e = 0; e < HD / 8; e++) x[e] = __builtin_fmaf(part[k][w][d0 + e], wt, x[e]);
            }
            const int i = v / G, hd = g * G + v - i * G, r = u.q0 + i;
            float* to;
            if (a.S == 1) {
                to = a.out + r * a.out_row + hd * a.out_head + d0;
            } else {
                const size_t rec = ((size_t)s * a.R + r) * a.NH + hd;
                to = a.po + rec * HD + d0;
                if (d0 == 0) *reinterpret_cast<sgpu_f32x4*>(a.pml + 4 * rec) = sgpu_f32x4{M, L, (float)used, 0.0f};
            }
#pragma unroll
            for (int e = 0; e < HD / 8; e += 4)
                *reinterpret_cast<sgpu_f32x4*>(to + e) = sgpu_f32x4{x[e], x[e + 1], x[e + 2], x[e + 3]};
        }
        __syncthreads();
    }
}

// The splits of each row and head joined, a wave each: 64 / T splits side by side, HD = 4 T dims.  The first
// split's record says how many there are.
template <int HD>
__device__ __forceinline__ void tree_join(const paged_tree& a) {
    constexpr int T = HD / 4, P = 64 / T;
    const int n = a.R * a.NH, t = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (t >= n) return;
    const int r = t / a.NH, hd = t - r * a.NH, lane = threadIdx.x & 63, part = lane / T, d = lane % T * 4;
    if (r < a.q_start[0] || r >= a.q_start[a.B]) return;
    const sgpu_f32x4* ml = reinterpret_cast<const sgpu_f32x4*>(a.pml);
    const int S = (int)ml[t][2];
    float M = -INFINITY, L = 0.0f;
    for (int s = lane; s < S; s += 64) M = fmaxf(M, ml[(size_t)s * n + t][0]);
    M = sgpu_wave_max(M);
    const float base = M == -INFINITY ? 0.0f : M;
    for (int s = lane; s < S; s += 64) {
        const sgpu_f32x4 y = ml[(size_t)s * n + t];
        L += y[1] * __builtin_amdgcn_exp2f(y[0] - base);
    }
    L = sgpu_wave_sum(L);
    sgpu_f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = part; s < S; s += P) {
        const sgpu_f32x4 y = ml[(size_t)s * n + t], v = *reinterpret_cast<const sgpu_f32x4*>(a.po + ((size_t)s * n + t) * HD + d);
        if (y[1] == 0.0f) continue;                   // this split saw nothing of the row
        const float w = y[1] * __builtin_amdgcn_exp2f(y[0] - base) / L;
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = __builtin_fmaf(v[e], w, x[e]);
    }
#pragma unroll
    for (int o = T; o < 64; o *= 2)
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] += __shfl_xor(x[e], o);
    if (part == 0) *reinterpret_cast<sgpu_f32x4*>(a.out + r * a.out_row + hd * a.out_head + d) = x;
}

// ---- logits ----
constexpr int kLogits = 8192;             // values of a block: eight a thread

// Row r's chunk c.  First the row's tokens that fall into the chunk are counted in LDS (whole numbers: their order
// does not matter), the latest of a token's biases found, and then each value is read, adjusted and written once.  What
// a penalty or bias touches is computed in 64 bits and rounded once.  In place, only what changes is read or written.
template <typename X, bool BIAS>
__device__ __forceinline__ void logits(const paged_logits& a) {
    __shared__ __attribute__((aligned(16))) uint32_t said[kLogits], last[BIAS ? kLogits : 4];
    typedef X vec __attribute__((ext_vector_type(8), aligned(sizeof(X))));
    const int tid = threadIdx.x, c = blockIdx.x % a.C, r = blockIdx.x / a.C;
    const int v0 = c * kLogits, n = min(kLogits, a.V - v0), e0 = 8 * tid;
    const X* const x = (const X*)a.x + r * a.x_row + v0 + e0;
    X* const y = (X*)a.y + r * a.y_row + v0 + e0;
    const bool same = a.x == a.y, whole = e0 + 8 <= n;
    vec in = {};
    if (!same && whole) in = *reinterpret_cast<const vec*>(x);
    uint32_t allow = 0xff;
    if (a.allow && e0 < n) allow = ((const uint8_t*)(a.allow + r * a.allow_row))[(v0 + e0) / 8];
    *reinterpret_cast<sgpu_u32x4*>(said + e0) = sgpu_u32x4{0, 0, 0, 0};
    *reinterpret_cast<sgpu_u32x4*>(said + e0 + 4) = sgpu_u32x4{0, 0, 0, 0};
    if constexpr (BIAS) {
        *reinterpret_cast<sgpu_u32x4*>(last + e0) = sgpu_u32x4{0, 0, 0, 0};
        *reinterpret_cast<sgpu_u32x4*>(last + e0 + 4) = sgpu_u32x4{0, 0, 0, 0};
    }
    __syncthreads();
    if (a.span) {
        // prompt: bit 31; output: counted
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const int from = min(max(a.span[4ll * r + 2 * k], 0), a.n_tok);
            const int to = from + min(max(a.span[4ll * r + 2 * k + 1], 0), a.n_tok - from);
            for (long long j = (long long)from + tid; j < to; j += 1024) {
                const uint32_t at = (uint32_t)a.tok[j] - (uint32_t)v0;
                if (a.tok[j] < 0 || at >= (uint32_t)n) continue;
                if (k == 0) atomicOr(&said[at], 0x80000000u);
                else atomicAdd(&said[at], 1u);
            }
        }
    }
    int b0 = 0;
    if constexpr (BIAS) {
        b0 = min(max(a.bias_span[2ll * r], 0), a.n_bias);
        const int nb = min(max(a.bias_span[2ll * r + 1], 0), a.n_bias - b0);
        for (int j = tid; j < nb; j += 1024) {
            const int id = a.bias_id[b0 + j];
            const uint32_t at = (uint32_t)id - (uint32_t)v0;
            if (id >= 0 && at < (uint32_t)n) atomicMax(&last[at], (uint32_t)j + 1u);
        }
    }
    __syncthreads();
    if (e0 >= n) return;
    uint32_t w[8], bi[8], any = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        w[j] = said[e0 + j];
        bi[j] = BIAS ? last[e0 + j] : 0;
        any |= w[j] | bi[j];
    }
    if (same && allow == 0xff && any == 0) return;
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    if (any) {
        if (a.rep) rep = a.rep[r];
        if (a.freq) freq = a.freq[r];
        if (a.pres) pres = a.pres[r];
    }
    vec out;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        if (!whole || same) in[j] = e0 + j < n ? x[j] : (X)0;
        out[j] = in[j];
        if (!(allow >> j & 1)) {
            out[j] = (X)-INFINITY;
        } else if (w[j] | bi[j]) {
            double z = (double)in[j];
            if (w[j]) z = z > 0.0 ? z / (double)rep : z * (double)rep;
            if (w[j] & 0x7fffffffu) z = z - (double)freq * (double)(w[j] & 0x7fffffffu) - (double)pres;
            if (bi[j]) z += (double)a.bias[b0 + (int)bi[j] - 1];
            out[j] = (X)z;
        }
    }
    if (whole) {
        *reinterpret_cast<vec*>(y) = out;
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (e0 + j < n) y[j] = out[j];
    }
}

}  // namespace

#define SGPU_HEADS(NAME, QO, KO, PAGED, VEC)                                                                          \
    extern "C" __global__ void __launch_bounds__(256) sgpu_heads_##NAME(paged_heads a) { heads<QO, KO, PAGED, VEC>(a); }
SGPU_HEADS(rows_f32, float, float, false, false)
SGPU_HEADS(rows_f16, _Float16, _Float16, false, false)
SGPU_HEADS(rows_v8_f32, float, float, false, true)
SGPU_HEADS(rows_v8_f16, _Float16, _Float16, false, true)
SGPU_HEADS(pages_f32, float, float, true, false)
SGPU_HEADS(pages_f16, float, _Float16, true, false)
SGPU_HEADS(pages_v8_f32, float, float, true, true)
SGPU_HEADS(pages_v8_f16, float, _Float16, true, true)

#define SGPU_TREE(HD)                                                                                                 \
    extern "C" __global__ void __launch_bounds__(256) sgpu_tree_f32_##HD(paged_tree a) { tree<HD, float>(a); }        \
    extern "C" __global__ void __launch_bounds__(256) sgpu_tree_f16_##HD(paged_tree a) { tree<HD, _Float16>(a); }     \
    extern "C" __global__ void __launch_bounds__(256) sgpu_tree_join_##HD(paged_tree a) { tree_join<HD>(a); }
SGPU_TREE(32)
SGPU_TREE(64)
SGPU_TREE(128)

#define SGPU_LOGITS(NAME, X, BIAS)                                                                                    \
    extern "C" __global__ void __launch_bounds__(1024) sgpu_logits_##NAME(paged_logits a) { logits<X, BIAS>(a); }
SGPU_LOGITS(f32, float, false)
SGPU_LOGITS(f16, _Float16, false)
SGPU_LOGITS(bias_f32, float, true)
SGPU_LOGITS(bias_f16, _Float16, true)
