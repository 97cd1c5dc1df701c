/* score.c -- launchers of sgpu_score.hip: rotary positions of rows, log probabilities, attention
 * over a shared prefix (part of libswitchgpu.so).  No reference counterpart. */
#include <math.h>
#include <string.h>

#include "sgpu_internal.h"
#include "switch_gpu.h"

/* rope: half / neighbouring pairs, one value or four a lane, fp32 or fp16 rows; then fp32 and fp16
 * logits, prefix caches by head size */
const char *const sgpu_score_kernels[SGPU_NSCORE] = {
    "sgpu_rope_rows_half_f32", "sgpu_rope_rows_half_f16", "sgpu_rope_rows_half_v4_f32", "sgpu_rope_rows_half_v4_f16",
    "sgpu_rope_rows_inter_f32", "sgpu_rope_rows_inter_f16", "sgpu_rope_rows_inter_v4_f32",
    "sgpu_rope_rows_inter_v4_f16",
    "sgpu_lp_part_f32", "sgpu_lp_part_f16", "sgpu_lp_join_f32", "sgpu_lp_join_f16",
#define ATTN_KERNELS(KIND) "sgpu_attn_" KIND "_32", "sgpu_attn_" KIND "_64", "sgpu_attn_" KIND "_128"
    ATTN_KERNELS("few_f32"), ATTN_KERNELS("few_f16"), ATTN_KERNELS("step_f32"), ATTN_KERNELS("rows_f32"),
    ATTN_KERNELS("rows_f16"), ATTN_KERNELS("cut_step"), ATTN_KERNELS("cut_rows"), ATTN_KERNELS("cut_prefix"),
    ATTN_KERNELS("join_few_f32"), ATTN_KERNELS("join_few_f16"), ATTN_KERNELS("join_many_f32"), ATTN_KERNELS("join_many_f16"),
};

static int misaligned(const void *p, size_t to) { return ((uintptr_t)p & (to - 1)) != 0; }

/* ---- rotary positions ---- */
int sgpu_rope_turns(const sgpu_rope_cfg *c, double *turns, float *mscale) {
    if (!c || !turns || c->rot < 2 || c->rot > SGPU_ROPE_MAX || c->rot % 2 || !(c->theta > 1.0) || isinf(c->theta) ||
        c->scaling < SGPU_ROPE_PLAIN || c->scaling > SGPU_ROPE_YARN)
        return SGPU_ERR_INVALID_ARG;
    const int bands = c->scaling == SGPU_ROPE_BANDS, yarn = c->scaling == SGPU_ROPE_YARN, rot = c->rot;
    if (c->scaling != SGPU_ROPE_PLAIN && (!(c->factor >= 1.0) || isinf(c->factor))) return SGPU_ERR_INVALID_ARG;
    if ((bands || yarn) && (!(c->ctx > 0.0) || isinf(c->ctx) || isinf(c->lo) || isinf(c->hi))) return SGPU_ERR_INVALID_ARG;
    if (bands && !(c->lo > 0.0 && c->hi > c->lo)) return SGPU_ERR_INVALID_ARG;
    if (yarn && !(c->hi > 0.0 && c->lo > c->hi)) return SGPU_ERR_INVALID_ARG;
    const double tau = 6.283185307179586476925;
    double theta = c->theta, first = 0.0, width = 1.0;
    if (c->scaling == SGPU_ROPE_BASE && rot > 2) theta *= pow(c->factor, (double)rot / (rot - 2));
    if (yarn) {                                  /* the ramp's first index and its length */
        const double fast = rot * log(c->ctx / (c->lo * tau)) / (2.0 * log(theta));
        const double slow = rot * log(c->ctx / (c->hi * tau)) / (2.0 * log(theta));
        first = fmax(floor(fast), 0.0);
        width = fmax(fmin(ceil(slow), rot - 1.0) - first, 1e-3);
    }
    for (int i = 0; i < rot / 2; i++) {
        const double f = pow(theta, -2.0 * i / rot);
        double w = 1.0;                          /* how much of f stays; the rest is divided by factor */
        if (c->scaling == SGPU_ROPE_LINEAR) w = 0.0;
        if (bands) w = fmin(1.0, fmax(0.0, (c->ctx * f / tau - c->lo) / (c->hi - c->lo)));
        if (yarn) w = 1.0 - fmin(1.0, fmax(0.0, (i - first) / width));
        turns[i] = (w == 1.0 ? f : f * w + f * (1.0 - w) / c->factor) / tau;
    }
    if (mscale) *mscale = yarn ? (float)(0.1 * log(c->factor) + 1.0) : 1.0f;
    return SGPU_OK;
}

#define ROPE_TABLE 2048        /* kRopeTable of sgpu_score.hip */
static int rope_rows(int half_out, const float *x, long long xs, void *y, long long ys, const int *pos, int pos0,
                     const double *turns, int rot, int neighbours, float mscale, int T, int H, int HD, void *stream) {
    if (T < 0 || T > 1 << 30 || H < 0 || HD < 1 || rot < 0 || rot % 2 || rot > SGPU_ROPE_MAX || rot > HD) return SGPU_ERR_INVALID_ARG;
    if (T == 0 || H == 0) return SGPU_OK;
    const long long n = (long long)H * HD;
    if (!x || !y || xs < n || ys < n || n > 1LL << 22 || (rot > 0 && !turns)) return SGPU_ERR_INVALID_ARG;
    if (misaligned(x, 4) || misaligned(y, half_out ? 2 : 4) || misaligned(pos, 4) || misaligned(turns, 8))
        return SGPU_ERR_INVALID_ARG;
    int same = (const void *)x == y;
    if (same && (xs != ys || half_out)) return SGPU_ERR_INVALID_ARG;
    if (same && rot == 0) return SGPU_OK;
    /* Rows of a block: enough values for its threads, within the table of angles. */
    int tb = 1;
    while (tb * n < 4096 && (long long)tb * rot < ROPE_TABLE && (long long)(T / (2 * tb)) >= 512) tb *= 2;
    const int vec = !misaligned(x, 16) && !misaligned(y, half_out ? 8 : 16) && xs % 4 == 0 && ys % 4 == 0 && HD % 4 == 0 &&
                    rot % (neighbours ? 4 : 8) == 0;
    void *args[] = {&x, &xs, &y, &ys, &pos, &pos0, &turns, &rot, &mscale, &T, &H, &HD, &tb, &same};
    const long long blocks = ((long long)T + tb - 1) / tb;
    return sgpu_internal_score_launch(SGPU_SC_ROPE + 4 * (neighbours != 0) + 2 * vec + half_out,
                                      (unsigned)(blocks < 1 << 20 ? blocks : 1 << 20), 256, args, stream);
}
int sgpu_rope_rows(const float *x, long long x_row, float *y, long long y_row, const int *pos, int pos0,
                   const double *turns, int rot, int neighbours, float mscale, int T, int H, int HD, void *stream) {
    return rope_rows(0, x, x_row, y, y_row, pos, pos0, turns, rot, neighbours, mscale, T, H, HD, stream);
}
int sgpu_rope_rows_h(const float *x, long long x_row, uint16_t *y, long long y_row, const int *pos, int pos0,
                     const double *turns, int rot, int neighbours, float mscale, int T, int H, int HD, void *stream) {
    return rope_rows(1, x, x_row, y, y_row, pos, pos0, turns, rot, neighbours, mscale, T, H, HD, stream);
}

/* ---- log probabilities ---- */
/* Chunks of a row: whole block tiles of 8192 values, and as few as fill the device. */
typedef struct {
    int C, len;
} lp_plan;
static int lp_sizes(int rows, int V, int k) {
    return rows > 0 && rows < 1 << 24 && V > 0 && k >= 0 && k <= SGPU_LOGPROBS_MAX_TOP && V <= 1 << 30;
}
static lp_plan lp_chunks(int rows, int V) {
    const int tiles = (V + 8191) / 8192;
    int C = 1024 / rows;
    if (C > tiles) C = tiles;
    if (C < 1) C = 1;
    const int per = (tiles + C - 1) / C;
    const lp_plan p = {(tiles + per - 1) / per, per * 8192};
    return p;
}
size_t sgpu_logprobs_workspace(int rows, int V, int k) {
    if (!lp_sizes(rows, V, k)) return 0;
    return (size_t)rows * (size_t)lp_chunks(rows, V).C * (16 + 8 * (size_t)k);
}
static int logprobs(int half, const void *x, long long xs, int rows, int V, const int *tok, int nt, float *logp,
                    float *entropy, int k, float *top_logp, int *top_id, void *ws, size_t ws_bytes, void *stream) {
    if (rows < 0 || nt < 0 || k < 0 || k > SGPU_LOGPROBS_MAX_TOP || V < 1) return SGPU_ERR_INVALID_ARG;
    if (rows == 0) return SGPU_OK;
    if (!lp_sizes(rows, V, k) || !x || xs < V || (nt > 0 && (!tok || !logp)) || (k > 0 && (!top_logp || !top_id)) || !ws ||
        misaligned(ws, 16) || misaligned(x, half ? 2 : 4) || ws_bytes < sgpu_logprobs_workspace(rows, V, k))
        return SGPU_ERR_INVALID_ARG;
    lp_plan p = lp_chunks(rows, V);
    float *part = (float *)ws;
    uint64_t *keys = (uint64_t *)(part + 4 * (size_t)rows * (size_t)p.C);
    void *a1[] = {&x, &xs, &V, &p.C, &p.len, &k, &part, &keys};
    int rc = sgpu_internal_score_launch(SGPU_SC_LP_PART + half, (unsigned)rows * (unsigned)p.C, 256, a1, stream);
    if (rc) return rc;
    void *a2[] = {&x, &xs, &V, &p.C, &tok, &nt, &logp, &entropy, &k, &top_logp, &top_id, &part, &keys};
    return sgpu_internal_score_launch(SGPU_SC_LP_JOIN + half, (unsigned)rows, 64, a2, stream);
}
int sgpu_logprobs(const float *x, long long x_row, int rows, int V, const int *tok, int nt, float *logp,
                  float *entropy, int k, float *top_logp, int *top_id, void *ws, size_t ws_bytes, void *stream) {
    return logprobs(0, x, x_row, rows, V, tok, nt, logp, entropy, k, top_logp, top_id, ws, ws_bytes, stream);
}
int sgpu_logprobs_h(const uint16_t *x, long long x_row, int rows, int V, const int *tok, int nt, float *logp,
                    float *entropy, int k, float *top_logp, int *top_id, void *ws, size_t ws_bytes, void *stream) {
    return logprobs(1, x, x_row, rows, V, tok, nt, logp, entropy, k, top_logp, top_id, ws, ws_bytes, stream);
}

/* ---- attention over a shared prefix ---- */
/* attn_prefix of sgpu_score.hip */
typedef struct {
    const void *q, *kp, *vp, *ks, *vs;
    float *out;
    const int *q_start, *kv_start, *kv_len;
    float *po, *pml;
    long long q_row, q_head, out_row, out_head, kp_row, kp_head, ks_row, ks_head;
    int R, B, P, SR, NH, NKV;
    float scale;
    int Sp, stages, step, run, MTp, nbp, nbs, MTs, Ss, wide_p, wide_s;
    uint16_t *cut;
    int *scales;
} attn_args;

static int stride_ok(long long row, long long head, int rows, int heads, long long quad) {
    return (rows <= 1 || (row > 0 && row <= SGPU_ATTN_PREFIX_MAX_ROW)) && (heads <= 1 || (head > 0 && head <= 1LL << 40)) &&
           row % quad == 0 && head % quad == 0;
}
/* The call's arguments but its workspace; SGPU_OK with R or B 0 is a call without work. */
static int attn_check(const sgpu_attn_prefix_args *a, int half) {
    if (!a || a->R < 0 || a->B < 0 || a->P < 0 || a->SR < 0 || a->NH <= 0 || a->NKV <= 0 || a->NH % a->NKV ||
        (a->HD != 32 && a->HD != 64 && a->HD != 128) || a->max_q < 0 || a->max_kv < 0 || !isfinite(a->scale) ||
        a->scale < 0.0f)
        return SGPU_ERR_INVALID_ARG;
    if (a->R == 0 || a->B == 0) return SGPU_OK;
    if ((long long)a->R * a->NH >= 1LL << 26 || (long long)a->B * a->NKV >= 1LL << 23) return SGPU_ERR_INVALID_ARG;
    if (!a->q || !a->out || !a->q_start || misaligned(a->q, 16) || misaligned(a->out, 16) || misaligned(a->q_start, 4) ||
        !stride_ok(a->q_row, a->q_head, a->R, a->NH, 4) || !stride_ok(a->out_row, a->out_head, a->R, a->NH, 4))
        return SGPU_ERR_INVALID_ARG;
    const long long quad = half ? 8 : 4;
    if (a->P > 0 && (!a->kp || !a->vp || misaligned(a->kp, 16) || misaligned(a->vp, 16) ||
                     !stride_ok(a->kp_row, a->kp_head, a->P, a->NKV, quad)))
        return SGPU_ERR_INVALID_ARG;
    if (a->SR > 0 && (!a->ks || !a->vs || misaligned(a->ks, 16) || misaligned(a->vs, 16) || !a->kv_start || !a->kv_len ||
                      misaligned(a->kv_start, 4) || misaligned(a->kv_len, 4) ||
                      !stride_ok(a->ks_row, a->ks_head, a->SR, a->NKV, quad)))
        return SGPU_ERR_INVALID_ARG;
    return SGPU_OK;
}
static int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }
static int imin(int a, int b) { return a < b ? a : b; }
static int imax(int a, int b) { return a > b ? a : b; }

/* The kernels of a call, by its rows: at most 32 a KV head (`few`: the waves of a block share the rows), more
 * (128 a block), and for fp32 keys that enough blocks read, those cut to fp16 pieces first.  `steps`: 64 keys of
 * a row tile, in all.  Both sides of the last rule, us (P prefix keys, HD 64 but where said):
 *    7896 steps (P  3001):  70 cut, 70 as they come;   7000 (P 32000):  75, 68;   8250 (P 24000):  77, 74
 *   10528 steps (P 12000):  89,     92;               11844 (P  3001):  89, 92;  15792 (P  3001): 113, 136
 *   HD 32,   7896 steps:    49,     52;   HD 128, 1316 steps:  59,  46;  2632:  72, 72;  5264: 98, 117 */
enum { ATTN_FEW_F32, ATTN_FEW_F16, ATTN_STEP_F32, ATTN_ROWS_F32, ATTN_ROWS_F16, ATTN_CUT_STEP, ATTN_CUT_ROWS, ATTN_CUT_PREFIX,
       ATTN_JOIN };
static int attn_cuts(int half, const sgpu_attn_prefix_args *a, const attn_args *k) {
    const long long steps = (long long)k->MTp * a->NKV * k->stages;
    return !half && k->wide_p && steps >= (a->HD <= 64 ? 8192 : 2560);
}

/* Row tiles, blocks and splits, from sizes and hints alone (the same on every device). */
static void attn_plan(int half, const sgpu_attn_prefix_args *a, attn_args *k) {
    const int G = a->NH / a->NKV, mq = imax(1, imin(a->max_q, a->R));
    const long long rp = (long long)a->R * G, rs = (long long)mq * G;
    k->wide_p = rp > 32;
    k->wide_s = k->wide_p && (half || rs > 32);
    k->MTp = ceil_div(rp, k->wide_p ? 128 : 32);
    const int room = (int)((1LL << 22) / ((long long)a->B * a->NKV));      /* (blocks take further tiles in turn) */
    k->MTs = imin(ceil_div(rs, k->wide_s ? 128 : 32), imax(1, room));
    /* Own keys: enough splits that every CU has two blocks. */
    k->Ss = 0;
    if (a->SR > 0) {
        const int want = imax(1, (int)(512 / ((long long)a->B * a->NKV * k->MTs)));
        k->Ss = imax(1, imin(imin(want, 16), ceil_div(imin(a->max_kv, a->SR), k->wide_s ? 128 : 256)));
    }
    /* The prefix: as many blocks as the CUs hold at once.  Short runs leave room for the own keys' blocks, so that
     * all start together.  A second step costs a block some 2 us, another split the join less: runs of one step in the
     * few-row form (4 rows of 14 heads, 500 keys: 8.0 + 4.8 us, 9.8 + 3.8 with two; 8000 keys: 8.3, 12.9) and,
     * with 128 rows, up to 8 steps in all (12 x 128 rows, 300 keys: 9.4 + 5.1, 12.5 + 4.3; 1000: 11.1 + 5.4, 11.6 + 4.2). */
    const long long units = (long long)k->MTp * a->NKV;
    k->step = k->wide_p ? 64 : 128;
    while (units * ceil_div(a->P, k->step) >= 1LL << 30) k->step *= 2;
    k->stages = ceil_div(a->P, k->step);
    const long long total = units * k->stages, own = (long long)a->B * a->NKV * k->MTs * k->Ss;
    const int cuts = attn_cuts(half, a, k);
    int slots = cuts && a->HD <= 64 ? 768 : cuts || half || a->HD <= 64 ? 512 : 256;
    if (!cuts && total < 8LL * slots) slots = (int)(own < slots / 2 ? slots - own : slots / 2);
    k->run = imax(k->wide_p && k->stages > 8 ? 2 : 1, ceil_div(total, slots));
    k->nbp = ceil_div(total, k->run);
    k->Sp = k->nbp > 0 ? imin(ceil_div(k->stages - 1, k->run) + 1, k->stages) : 0;
}
static size_t attn_workspace(int half, const sgpu_attn_prefix_args *a, const attn_args *k) {
    const size_t n = (size_t)a->R * (size_t)a->NH;
    size_t bytes = (size_t)(k->Sp + k->Ss) * n * ((size_t)a->HD + 4) * sizeof(float) + 16;
    if (attn_cuts(half, a, k)) bytes += (size_t)a->NKV * ((size_t)a->P * a->HD * 8 + ((size_t)a->P + 31) / 32 * 16);
    return bytes;
}
size_t sgpu_attn_prefix_workspace(const sgpu_attn_prefix_args *a) {
    attn_args k, h;
    if (attn_check(a, 0) || a->R == 0 || a->B == 0) return 0;
    attn_plan(0, a, &k);
    attn_plan(1, a, &h);
    const size_t f32 = attn_workspace(0, a, &k), f16 = attn_workspace(1, a, &h);
    return f32 > f16 ? f32 : f16;
}
static int attn_launch(int kernel, const sgpu_attn_prefix_args *a, long long blocks, attn_args *k, void *stream) {
    void *args[] = {k};
    const int j = a->HD == 32 ? 0 : a->HD == 64 ? 1 : 2;
    return blocks > 0 ? sgpu_internal_score_launch(SGPU_SC_ATTN + 3 * kernel + j, (unsigned)blocks, 256, args, stream) : SGPU_OK;
}
static int attn_prefix(int half, const sgpu_attn_prefix_args *a, void *ws, size_t ws_bytes, void *stream) {
    int rc = attn_check(a, half);
    if (rc || a->R == 0 || a->B == 0) return rc;
    attn_args k = {a->q, a->kp, a->vp, a->ks, a->vs, a->out, a->q_start, a->kv_start, a->kv_len, NULL, NULL,
                   a->q_row, a->q_head, a->out_row, a->out_head, a->kp_row, a->kp_head, a->ks_row, a->ks_head,
                   a->R, a->B, a->P, a->SR, a->NH, a->NKV, a->scale, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, NULL, NULL};
    attn_plan(half, a, &k);
    const int S = k.Sp + k.Ss;
    const long long n = (long long)a->R * a->NH, own = k.Ss ? (long long)a->B * a->NKV * k.MTs * k.Ss : 0;
    if (!ws || misaligned(ws, 16) || ws_bytes < attn_workspace(half, a, &k)) return SGPU_ERR_INVALID_ARG;
    k.nbs = (int)own;
    k.po = (float *)ws;
    k.pml = k.po + (size_t)S * (size_t)n * a->HD;
    if (attn_cuts(half, a, &k)) {
        const int grps = ceil_div(a->P, 32);
        k.scales = (int *)(k.pml + 4 * (size_t)S * (size_t)n);
        k.cut = (uint16_t *)(k.scales + (size_t)a->NKV * grps * 4);
        rc = attn_launch(k.wide_s ? ATTN_CUT_ROWS : ATTN_CUT_STEP, a, own + ceil_div((long long)a->NKV * grps, 4), &k,
                         stream);
        if (!rc) rc = attn_launch(ATTN_CUT_PREFIX, a, k.nbp, &k, stream);
    } else {
        const int kernel = half ? (k.wide_p ? ATTN_ROWS_F16 : ATTN_FEW_F16)
                                : k.wide_s ? ATTN_ROWS_F32 : k.wide_p ? ATTN_STEP_F32 : ATTN_FEW_F32;
        rc = attn_launch(kernel, a, k.nbp + own, &k, stream);
    }
    if (rc) return rc;
    /* a wave a row where it has many splits, else HD / 4 lanes */
    const int many = S > 8;
    return attn_launch(ATTN_JOIN + 2 * many + half, a, ceil_div(n * (many ? 64 : a->HD / 4), 256), &k, stream);
}
int sgpu_attn_prefix(const sgpu_attn_prefix_args *a, void *ws, size_t ws_bytes, void *stream) {
    return attn_prefix(0, a, ws, ws_bytes, stream);
}
int sgpu_attn_prefix_h(const sgpu_attn_prefix_args *a, void *ws, size_t ws_bytes, void *stream) {
    return attn_prefix(1, a, ws, ws_bytes, stream);
}
