// sgpu_score.hip -- what a host that scores or samples several continuations of one prompt needs
// beside the decode engines' own kernels (gfx950):
//   sgpu_rope_rows_*    rotary positions of rows at positions of their own
//   sgpu_logprobs_*     log probabilities of given tokens, entropy and top alternatives of logits
//   sgpu_attn_prefix_*  attention of a batch whose sequences share a long prefix
// fp16 values here are IEEE ones (infinities, NaN and subnormals as they are), unlike the weight
// codes of the GEMVs.
#include "sgpu_device.h"

namespace {

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_a2 __attribute__((ext_vector_type(8), aligned(2)));

// ---- rotary positions ----
// sin and cos of 2 pi u, u in turns: u is reduced to the nearest quarter turn in 64 bits (a far
// position's angle has no fp32 digits left), the rest, at most an eighth of a turn, goes through
// the Taylor series of both (first term left out below 2e-9 of 1).
__device__ __forceinline__ void sincos_turns(double u, float& sn, float& cs) {
    const double quarters = rint(4.0 * u);
    const float x = (float)((u - 0.25 * quarters) * 6.283185307179586476925), x2 = x * x;
    float s = __builtin_fmaf(x2, 2.7557319e-6f, -1.98412698e-4f);
    s = __builtin_fmaf(s, x2, 8.33333333e-3f);
    s = __builtin_fmaf(s, x2, -0.166666667f);
    s = __builtin_fmaf(s * x2, x, x);
    float c = __builtin_fmaf(x2, -2.75573192e-7f, 2.48015873e-5f);
    c = __builtin_fmaf(c, x2, -1.38888889e-3f);
    c = __builtin_fmaf(c, x2, 4.16666667e-2f);
    c = __builtin_fmaf(c, x2, -0.5f);
    c = __builtin_fmaf(c, x2, 1.0f);
    const int q = (int)(quarters - 4.0 * floor(0.25 * quarters));       // 0..3
    sn = q & 1 ? c : s;
    cs = q & 1 ? s : c;
    if (q & 2) sn = -sn;
    if (q == 1 || q == 2) cs = -cs;
}

template <typename O> __device__ __forceinline__ void put4(O* p, const float (&v)[4]);
template <> __device__ __forceinline__ void put4<float>(float* p, const float (&v)[4]) {
    *reinterpret_cast<sgpu_f32x4*>(p) = sgpu_f32x4{v[0], v[1], v[2], v[3]};
}
template <> __device__ __forceinline__ void put4<_Float16>(_Float16* p, const float (&v)[4]) {
    *reinterpret_cast<f16x4*>(p) = f16x4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
}

constexpr int kRopeTable = 2048;      // (cos, sin) pairs a block holds: its rows by rot / 2

// Rows t of x (H heads of HD values, row stride xs) at position pos0 + (pos ? pos[t] : t), rotated
// into y (row stride ys): pair i of a head by turns[i] per position, pairs (i, i + rot/2) or
// (INTER) (2i, 2i + 1); values past rot pass through.  A block takes tb rows: the angles of its
// rows once into LDS, then every head reads them.  VEC: four values a lane and access (rows 16-byte
// aligned, HD, rot and rot/2 whole quads); otherwise a pair or one value a lane.
// Bound: the rows' way through memory; below some hundred rows the launch.
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

constexpr int kTop = 64;               // the most alternatives of a row

// Top alternatives of what one wave sees: `best`, its k best keys so far (LDS, 0 where none), and
// behind them `n` candidates that beat the k-th.  flush() ranks all of them by counting.
struct top_list {
    unsigned long long* best;          // kTop + 128 keys
    int k, n;
    unsigned long long kth;
};
__device__ __forceinline__ void lds_sync() {      // the wave's own LDS writes are seen by its other lanes
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
__device__ __forceinline__ void top_flush(top_list& l) {
    const int lane = threadIdx.x & 63, E = l.k + l.n;
    lds_sync();
    unsigned long long mine[3];
    int rank[3] = {0, 0, 0};
#pragma unroll
    for (int r = 0; r < 3; r++) mine[r] = lane + 64 * r < E ? l.best[lane + 64 * r] : 0;
    for (int i = 0; i < E; i++) {
        const unsigned long long o = l.best[i];
#pragma unroll
        for (int r = 0; r < 3; r++) rank[r] += o > mine[r];
    }
    lds_sync();
    // empty places share a rank past all keys and are written as empty
    for (int i = lane; i < l.k; i += 64) l.best[i] = 0;
    lds_sync();
#pragma unroll
    for (int r = 0; r < 3; r++)
        if (mine[r] && rank[r] < l.k) l.best[rank[r]] = mine[r];
    lds_sync();
    l.n = 0;
    l.kth = l.best[l.k - 1];
}
__device__ __forceinline__ void top_add(top_list& l, bool in, unsigned long long key) {
    const unsigned long long b = __ballot(in);
    if (!b) return;
    const int lane = threadIdx.x & 63;
    if (in) l.best[l.k + l.n + __popcll(b & ((1ull << lane) - 1))] = key;
    l.n += __popcll(b);
    if (l.n >= 64) top_flush(l);
}

template <typename X> struct logits;
template <> struct logits<float> {
    static constexpr int VEC = 4;
    __device__ static __forceinline__ void load(const float* p, float* v) {
        const sgpu_f32x4 a = sgpu_ld4<false>(p);
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = a[j];
    }
};
template <> struct logits<_Float16> {
    static constexpr int VEC = 8;
    __device__ static __forceinline__ void load(const _Float16* p, float* v) {
        const f16x8 a = *reinterpret_cast<const f16x8_a2*>(p);
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = (float)a[j];
    }
};

constexpr int kLpTile = 32;            // values a lane holds at a time

// Chunk c of row r (V values, C chunks of `len`): its statistics to part[(r * C + c) * 4 ..], its k
// best keys to keys[(r * C + c) * k ..].  256 threads; a wave takes tiles of 64 * kLpTile values.
template <typename X>
__device__ __forceinline__ void lp_part(const X* __restrict__ x, long long xs, int V, int C, int len, int k,
                                        float* __restrict__ part, unsigned long long* __restrict__ keys) {
    constexpr int VEC = logits<X>::VEC, NV = kLpTile / VEC;
    __shared__ unsigned long long lists[4][kTop + 128];
    __shared__ stats red[4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = blockIdx.x % C, r = blockIdx.x / C;
    const X* row = x + (long long)r * xs;
    const int v0 = c * len, v1 = min(V, v0 + len);
    top_list top = {lists[wave], k, 0, 0};
    for (int i = lane; i < k; i += 64) top.best[i] = 0;
    stats a = {-3.402823466e38f, 0.0f, 0.0f};
    for (int t0 = v0 + wave * 64 * kLpTile; t0 < v1; t0 += 4 * 64 * kLpTile) {
        float v[kLpTile];
        if (t0 + 64 * kLpTile <= v1) {
#pragma unroll
            for (int j = 0; j < NV; j++) logits<X>::load(row + t0 + (j * 64 + lane) * VEC, v + j * VEC);
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
        stats b = {mn, e0 * a.s, e0 > 0.0f ? e0 * __builtin_fmaf(d, a.s, a.w) : 0.0f};
#pragma unroll
        for (int j = 0; j < kLpTile; j++) {
            const float y = (v[j] - mn) * kLog2e, e = __builtin_amdgcn_exp2f(y);
            b.s += e;
            b.w = __builtin_fmaf(e, fmaxf(y, -256.0f), b.w);     // no weight, no part: 0 times an infinity
        }
        a = b;
        if (k > 0) {
            // Candidates: what beats the wave's k-th so far, and is not below the k-th largest of the
            // lanes' maxima (at least k values of this tile are no smaller), whose upper 16 bits a
            // binary search over the lanes finds.
            uint32_t from = (uint32_t)(top.kth >> 32);
            if (!__any(!(m <= value_of(from)))) continue;
            const uint32_t mo = order_of(m);
            uint32_t p = 0;
            for (uint32_t bit = 1u << 31; bit >= 1u << 16; bit >>= 1)
                if (__popcll(__ballot(mo >= (p | bit))) >= k) p |= bit;
            if (p > 0 && p - 1 > from) from = p - 1;
            const float f = value_of(from == 0x7fffffffu ? 0x7ffffffeu : from);      // no -0: it would equal +0
            uint32_t in = 0;
#pragma unroll
            for (int j = 0; j < kLpTile; j++) in |= !(v[j] <= f) ? 1u << j : 0u;
            while (__any(in != 0)) {               // mostly one or two a lane: read again, not kept by a register index
                const int j = in ? __builtin_ctz(in) : 0;
                const int i = t0 + ((j / VEC) * 64 + lane) * VEC + j % VEC;
                const bool ok = in != 0 && i < v1;
                const unsigned long long key = ok ? key_of((float)row[i], i) : 0;
                top_add(top, key > top.kth, key);
                in &= in - 1;
            }
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        stats b = {__shfl_xor(a.m, o), __shfl_xor(a.s, o), __shfl_xor(a.w, o)};
        join(a, b);
    }
    if (lane == 0) red[wave] = a;
    if (k > 0) top_flush(top);
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
        for (int w = 1; w < 4; w++) {
            const unsigned long long key = lane < k ? lists[w][lane] : 0;
            top_add(top, key > top.kth, key);
        }
        top_flush(top);
        if (lane < k) keys[u * k + lane] = top.best[lane];
    }
}

// Row r's results from its C parts: 64 threads.
template <typename X>
__device__ __forceinline__ void lp_join(const X* __restrict__ x, long long xs, int V, int C, const int* __restrict__ tok,
                                        int nt, float* __restrict__ logp, float* __restrict__ entropy, int k,
                                        float* __restrict__ top_logp, int* __restrict__ top_id,
                                        const float* __restrict__ part, const unsigned long long* __restrict__ keys) {
    __shared__ unsigned long long list[kTop + 128];
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
    top_list top = {list, k, 0, 0};
    for (int i = lane; i < k; i += 64) list[i] = 0;
    const unsigned long long* kr = keys + (size_t)r * C * k;
    for (int i0 = 0; i0 < C * k; i0 += 64) {
        const unsigned long long key = i0 + lane < C * k ? kr[i0 + lane] : 0;
        top_add(top, key > top.kth, key);
    }
    top_flush(top);
    if (lane < k) {
        const unsigned long long key = list[lane];
        top_id[(size_t)r * k + lane] = key && !odd ? (int)~(uint32_t)key : -1;
        top_logp[(size_t)r * k + lane] = odd ? a.s : key ? lp(value_of((uint32_t)(key >> 32))) : -INFINITY;
    }
}

// ---- attention over a shared prefix ----
}  // namespace

// What the launcher passes by value (sgpu_attn_prefix_args, include/switch_gpu.h, without its hints).
struct attn_prefix {
    const void *q, *kp, *vp, *ks, *vs;
    float* out;
    const int *q_start, *kv_start, *kv_len;
    long long q_row, q_head, out_row, out_head, kp_row, kp_head, ks_row, ks_head;
    int R, B, P, SR, NH, NKV;
    float scale;
};

namespace {

// Row r's sequence: its own keys' first row and how many of them the row sees; false for a row
// of no sequence.  Starts and lengths out of range are cut to it.
__device__ __forceinline__ bool row_keys(const attn_prefix& a, int r, int& first, int& seen) {
    int lo = 0, hi = a.B;                      // q_start[lo] <= r < q_start[hi]
    if (r < a.q_start[0] || r >= a.q_start[a.B]) return false;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (a.q_start[mid] <= r) lo = mid;
        else hi = mid;
    }
    first = seen = 0;
    if (a.SR == 0) return true;
    const int q0 = max(a.q_start[lo], 0), q1 = min(a.q_start[lo + 1], a.R);
    first = min(max(a.kv_start[lo], 0), a.SR);
    const int len = min(max(a.kv_len[lo], 0), a.SR - first);
    seen = min(max(len - (q1 - q0) + (r - q0) + 1, 0), len);
    return true;
}

// One wave a row and head, 64 keys at a time: a key a lane for the scores, then a dim (HD 128: two)
// a lane for the values.
template <int HD, typename KV>
__device__ __forceinline__ void attn_rows(const attn_prefix& a) {
    constexpr int ND = HD > 64 ? 2 : 1;
    __shared__ float qs[HD], ps[64];
    const int lane = threadIdx.x, r = blockIdx.x / a.NH, h = blockIdx.x % a.NH, g = h / (a.NH / a.NKV);
    int first, seen;
    if (!row_keys(a, r, first, seen)) return;
    const float* q = (const float*)a.q + r * a.q_row + h * a.q_head;
    for (int d = lane; d < HD; d += 64) qs[d] = q[d];
    lds_sync();
    float m = -INFINITY, l = 0.0f, o[ND];
    for (int e = 0; e < ND; e++) o[e] = 0.0f;
    for (int part = 0; part < 2; part++) {
        const int n = part ? seen : a.P;
        const long long row = part ? a.ks_row : a.kp_row;
        const KV* K = (part ? (const KV*)a.ks + first * row + g * a.ks_head : (const KV*)a.kp + g * a.kp_head);
        const KV* W = (part ? (const KV*)a.vs + first * row + g * a.ks_head : (const KV*)a.vp + g * a.kp_head);
        for (int j0 = 0; j0 < n; j0 += 64) {
            float s = 0.0f;
            const KV* kr = K + min(j0 + lane, n - 1) * row;
            for (int d = 0; d < HD; d++) s = __builtin_fmaf(qs[d], (float)kr[d], s);
            s = j0 + lane < n ? s * a.scale * kLog2e : -INFINITY;
            const float mn = fmaxf(m, sgpu_wave_max(s)), base = mn == -INFINITY ? 0.0f : mn;
            const float al = __builtin_amdgcn_exp2f(m - base), p = __builtin_amdgcn_exp2f(s - base);
            m = mn;
            l = l * al + sgpu_wave_sum(p);
            ps[lane] = p;
            lds_sync();
            for (int e = 0; e < ND; e++) {
                const int d = lane + 64 * e;
                float acc = o[e] * al;
                if (d < HD)
                    for (int j = 0; j < min(64, n - j0); j++) acc = __builtin_fmaf(ps[j], (float)W[(j0 + j) * row + d], acc);
                o[e] = acc;
            }
            lds_sync();
        }
    }
    for (int e = 0; e < ND; e++) {
        const int d = lane + 64 * e;
        if (d < HD) a.out[r * a.out_row + h * a.out_head + d] = l > 0.0f ? o[e] / l : l == 0.0f ? 0.0f : l;
    }
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

#define SGPU_ATTN_PREFIX(HD)                                                                                          \
    extern "C" __global__ void __launch_bounds__(64) sgpu_attn_prefix_f32_##HD(attn_prefix a) { attn_rows<HD, float>(a); } \
    extern "C" __global__ void __launch_bounds__(64) sgpu_attn_prefix_f16_##HD(attn_prefix a) { attn_rows<HD, _Float16>(a); }
SGPU_ATTN_PREFIX(32)
SGPU_ATTN_PREFIX(64)
SGPU_ATTN_PREFIX(128)
