/* paged.c -- launchers of sgpu_paged.hip: norms and rotations of heads, appending to a paged cache, attention of
 * new rows over pages, adjusting logits (part of libswitchgpu.so).  No reference counterpart. */
#include <math.h>
#include <string.h>

#include "sgpu_internal.h"
#include "switch_gpu.h"

/* heads: into rows or pages, one value or eight a lane, and of many rows, by output type; then attention by rows a block and
 * head size; logits without and with biases */
const char *const sgpu_paged_kernels[SGPU_NPAGED] = {
    "sgpu_heads_rows_f32", "sgpu_heads_rows_f16", "sgpu_heads_rows_v8_f32", "sgpu_heads_rows_v8_f16", "sgpu_heads_rows_v8s_f32",
    "sgpu_heads_rows_v8s_f16", "sgpu_heads_pages_f32", "sgpu_heads_pages_f16", "sgpu_heads_pages_v8_f32", "sgpu_heads_pages_v8_f16",
    "sgpu_heads_pages_v8s_f32", "sgpu_heads_pages_v8s_f16",
#define TREE_KERNELS(KIND) "sgpu_tree_" KIND "_32", "sgpu_tree_" KIND "_64", "sgpu_tree_" KIND "_128"
    TREE_KERNELS("r16_f32"), TREE_KERNELS("r32_f32"), TREE_KERNELS("r64_f32"), TREE_KERNELS("r128_f32"),
    TREE_KERNELS("r16_f16"), TREE_KERNELS("r32_f16"), TREE_KERNELS("r64_f16"), TREE_KERNELS("r128_f16"), TREE_KERNELS("join"),
    "sgpu_logits_f32", "sgpu_logits_f16", "sgpu_logits_bias_f32", "sgpu_logits_bias_f16",
};

static int misaligned(const void *p, size_t to) { return ((uintptr_t)p & (to - 1)) != 0; }
static int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }
static int imin(int a, int b) { return a < b ? a : b; }
static int imax(int a, int b) { return a > b ? a : b; }

/* A cache's description; `to`: what its addresses and strides are whole multiples of, in bytes, values of `size`. */
static int cache_ok(const sgpu_paged_kv *c, int NKV, size_t to, size_t size) {
    if (c->R < 0 || c->B < 0 || c->pages < 0 || c->page < 1 || c->table_pages < 0 ||
        (long long)c->table_pages * c->page > 1LL << 30)
        return 0;
    if (c->R == 0 || c->B == 0) return 1;
    if (!c->len || !c->q_start || misaligned(c->len, 4) || misaligned(c->q_start, 4)) return 0;
    if (c->pages == 0 || c->table_pages == 0) return 1;                /* no token has a place */
    const long long quad = (long long)(to / size), far = 1LL << 46;
    const long long s[3] = {c->page_stride, c->kv_row, c->kv_head}, n[3] = {c->pages, c->page, NKV};
    for (int i = 0; i < 3; i++)
        if (n[i] > 1 && (s[i] <= 0 || s[i] > far / n[i] || s[i] % quad)) return 0;
    return c->k && c->v && !misaligned(c->k, to) && !misaligned(c->v, to) && c->table && !misaligned(c->table, 4) &&
           (c->B == 1 || (c->table_row >= c->table_pages && c->table_row <= far / c->B));
}

/* ---- norms and rotations of heads ---- */
/* paged_heads of sgpu_paged.hip */
typedef struct {
    const float *q, *k, *v;
    void *yq, *yk, *yv;
    const float *wq, *wk;
    const int *pos;
    const double *turns;
    const int *table, *len, *q_start;
    long long q_row, k_row, v_row, yq_row, yk_row, table_row, page_stride, kv_row, kv_head;
    int pos0, rot, neighbours;
    float mscale, eps;
    double per;
    int T, NH, NKV, HD, tb, team;
    int pages, page, table_pages, B;
} heads_args;

static int heads_ok(int T, int NH, int NKV, int HD, int rot, const double *turns, float eps) {
    return T >= 0 && T <= 1 << 30 && NH >= 0 && NKV >= 0 && HD >= 1 && ((long long)NH + 2LL * NKV) * HD <= 1LL << 22 && rot >= 0 &&
           rot % 2 == 0 && rot <= SGPU_ROPE_MAX && rot <= HD && (rot == 0 || (turns && !misaligned(turns, 8))) &&
           isfinite(eps) && eps >= 0.0f;
}
/* vec: addresses and strides are whole quads of values. */
static int heads_launch(int kernel, heads_args *a, int vec, void *stream) {
    const int n = (a->NH + 2 * a->NKV) * a->HD;
    vec = vec && a->HD % 8 == 0 && a->HD <= 512 && a->rot % 8 == 0 && !misaligned(a->wq, 16) && !misaligned(a->wk, 16);
    a->per = 1.0 / a->HD;
    /* Rows of more than 64 MiB are read and written past the caches' usual order (84 MB of them 29.1 -> 26.3 us, 135 MB
     * 53.8 -> 49.3); smaller ones are often there still (20 MB 8.3, 9.4 past it). */
    const int once = vec && (long long)a->T * n > 16LL << 20;
    while (a->team < 6 && (8 << a->team) < a->HD) a->team++;
    /* Rows of a block: enough values for its threads, within the tables of places and angles. */
    a->tb = 1;
    while (a->tb < 64 && a->tb * n < 4096 && a->tb * a->rot <= 2048 && a->T / (2 * a->tb) >= 512) a->tb *= 2;
    void *args[] = {a};
    return sgpu_internal_paged_launch(SGPU_PG_HEADS + kernel + 2 * (vec + once), (unsigned)imin(ceil_div(a->T, a->tb), 1 << 20), 256, args,
                                      stream);
}
static int qk_norm_rope(int half_out, const float *x, long long x_row, void *y, long long y_row, const float *wq, const float *wk,
                        float eps, const int *pos, int pos0, const double *turns, int rot, int neighbours, float mscale, int T,
                        int NH, int NKV, int HD, void *stream) {
    if (!heads_ok(T, NH, NKV, HD, rot, turns, eps)) return SGPU_ERR_INVALID_ARG;
    const long long n = ((long long)NH + NKV) * HD;
    if (T == 0 || n == 0) return SGPU_OK;
    const size_t size = half_out ? 2 : 4;
    if (!x || !y || x_row < n || y_row < n || misaligned(x, 4) || misaligned(y, size) || misaligned(pos, 4) || misaligned(wq, 4) ||
        misaligned(wk, 4) || ((const void *)x == y && (half_out || x_row != y_row)))
        return SGPU_ERR_INVALID_ARG;
    heads_args a;
    memset(&a, 0, sizeof a);
    a.q = x; a.k = x + (long long)NH * HD;
    a.yq = y; a.yk = (char *)y + (size_t)NH * (size_t)HD * size;
    a.wq = wq; a.wk = wk; a.pos = pos; a.turns = turns;
    a.q_row = a.k_row = x_row; a.yq_row = a.yk_row = y_row;
    a.pos0 = pos0; a.rot = rot; a.neighbours = neighbours != 0; a.mscale = mscale; a.eps = eps;
    a.T = T; a.NH = NH; a.NKV = NKV; a.HD = HD;
    return heads_launch(half_out, &a, !misaligned(x, 16) && !misaligned(y, 4 * size) && x_row % 4 == 0 && y_row % 4 == 0, stream);
}
int sgpu_qk_norm_rope(const float *x, long long x_row, float *y, long long y_row, const float *wq, const float *wk, float eps,
                      const int *pos, int pos0, const double *turns, int rot, int neighbours, float mscale, int T, int NH,
                      int NKV, int HD, void *stream) {
    return qk_norm_rope(0, x, x_row, y, y_row, wq, wk, eps, pos, pos0, turns, rot, neighbours, mscale, T, NH, NKV, HD, stream);
}
int sgpu_qk_norm_rope_h(const float *x, long long x_row, uint16_t *y, long long y_row, const float *wq, const float *wk, float eps,
                        const int *pos, int pos0, const double *turns, int rot, int neighbours, float mscale, int T, int NH,
                        int NKV, int HD, void *stream) {
    return qk_norm_rope(1, x, x_row, y, y_row, wq, wk, eps, pos, pos0, turns, rot, neighbours, mscale, T, NH, NKV, HD, stream);
}

static int kv_append(int half, const sgpu_kv_append_args *p, void *stream) {
    if (!p) return SGPU_ERR_INVALID_ARG;
    const sgpu_paged_kv *c = &p->c;
    const size_t size = half ? 2 : 4;
    const int NH = p->q ? p->NH : 0, NKV = p->NKV, HD = p->HD;
    if (p->NH < 0 || NKV < 1 || !heads_ok(c->R, NH, NKV, HD, p->rot, p->turns, p->eps) || !cache_ok(c, NKV, size, size))
        return SGPU_ERR_INVALID_ARG;
    if (c->R == 0 || c->B == 0) return SGPU_OK;
    const long long n = (long long)NKV * HD, nq = (long long)NH * HD;
    if (!p->k || !p->v || p->k_row < n || p->v_row < n || misaligned(p->k, 4) || misaligned(p->v, 4) || misaligned(p->pos, 4) ||
        misaligned(p->wq, 4) || misaligned(p->wk, 4))
        return SGPU_ERR_INVALID_ARG;
    if (NH > 0 && (!p->q_out || misaligned(p->q, 4) || misaligned(p->q_out, 4) || p->q_row < nq || p->out_row < nq ||
                   (p->q == p->q_out && p->q_row != p->out_row)))
        return SGPU_ERR_INVALID_ARG;
    heads_args a;
    memset(&a, 0, sizeof a);
    a.q = p->q; a.k = p->k; a.v = p->v; a.yq = p->q_out; a.yk = c->k; a.yv = c->v;
    a.wq = p->wq; a.wk = p->wk; a.pos = p->pos; a.turns = p->turns;
    a.table = c->table; a.len = c->len; a.q_start = c->q_start;
    a.q_row = p->q_row; a.k_row = p->k_row; a.v_row = p->v_row; a.yq_row = p->out_row;
    a.table_row = c->table_row; a.page_stride = c->page_stride; a.kv_row = c->kv_row; a.kv_head = c->kv_head;
    a.rot = p->rot; a.neighbours = p->neighbours != 0; a.mscale = p->mscale; a.eps = p->eps;
    a.T = c->R; a.NH = NH; a.NKV = NKV; a.HD = HD;
    a.pages = c->pages; a.page = c->page; a.table_pages = c->pages ? c->table_pages : 0; a.B = c->B;
    int vec = !misaligned(p->k, 16) && !misaligned(p->v, 16) && p->k_row % 4 == 0 && p->v_row % 4 == 0 &&
              !misaligned(c->k, 4 * size) && !misaligned(c->v, 4 * size) && c->page_stride % 4 == 0 && c->kv_row % 4 == 0 &&
              c->kv_head % 4 == 0;
    if (NH > 0) vec = vec && !misaligned(p->q, 16) && !misaligned(p->q_out, 16) && p->q_row % 4 == 0 && p->out_row % 4 == 0;
    return heads_launch(6 + half, &a, vec, stream);
}
int sgpu_kv_append(const sgpu_kv_append_args *a, void *stream) { return kv_append(0, a, stream); }
int sgpu_kv_append_h(const sgpu_kv_append_args *a, void *stream) { return kv_append(1, a, stream); }

/* ---- attention over pages ---- */
/* paged_tree and tree_front of sgpu_paged.hip */
typedef struct {
    const void *k, *v;
    const float *q;
    float *out;
    const int *table;
    const uint32_t *mask;
    float *po, *pml;
    int *desc;
    long long page_stride, kv_row, kv_head, table_row, q_row, q_head, out_row, out_head, mask_row;
    int pages, page, table_pages, NH;
    float scale;
    int MT, shift, halves;
} tree_args;
typedef struct {
    int NB, MT, start, wide;                      /* wide: 16 << wide rows a block */
} tree_shape;

static int stride_ok(long long row, long long head, int rows, int heads) {
    return (rows <= 1 || (row > 0 && row <= 1LL << 40)) && (heads <= 1 || (head > 0 && head <= 1LL << 40)) && row % 4 == 0 && head % 4 == 0;
}
static int tree_check(const sgpu_attn_tree_args *a, int half) {
    if (!a || a->NH <= 0 || a->NKV <= 0 || a->NH % a->NKV || (a->HD != 32 && a->HD != 64 && a->HD != 128) || a->max_q < 0 ||
        a->max_kv < 0 || !isfinite(a->scale) || a->scale < 0.0f || !cache_ok(&a->c, a->NKV, 16, half ? 2 : 4))
        return SGPU_ERR_INVALID_ARG;
    if (a->c.R == 0 || a->c.B == 0) return SGPU_OK;
    if ((long long)a->c.R * a->NH >= 1LL << 26 || (long long)a->c.B * a->NKV >= 1LL << 23) return SGPU_ERR_INVALID_ARG;
    if (!a->q || !a->out || misaligned(a->q, 16) || misaligned(a->out, 16) || !stride_ok(a->q_row, a->q_head, a->c.R, a->NH) ||
        !stride_ok(a->out_row, a->out_head, a->c.R, a->NH))
        return SGPU_ERR_INVALID_ARG;
    if (a->mask && (misaligned(a->mask, 4) || a->mask_row < 0 || a->mask_row > 1 << 26)) return SGPU_ERR_INVALID_ARG;
    return SGPU_OK;
}
/* Rows a block and blocks, from sizes and hints alone (the same on every device).  Where a block for each row tile of a
 * sequence and KV head would not fill the device, the batch's steps are dealt out evenly instead (tree_line in
 * sgpu_paged.hip), to as many blocks as the CUs hold. */
static void tree_plan(int half, const sgpu_attn_tree_args *a, tree_shape *k) {
    const int G = a->NH / a->NKV, rows = imax(1, imin(a->max_q, a->c.R)) * G, room = a->c.pages ? a->c.table_pages * a->c.page : 0;
    const long long units = (long long)a->c.B * a->NKV;
    /* The smallest tile that takes a sequence's rows.  32 sequences of 3000 tokens, fp16, 2 KV heads of 64: 14 rows 16.4 us in
     * 16, 17.2 in 32; 28 rows 19.0 in 16, 18.1 in 32, 19.9 in 64; 112 rows 29.3 in 64, 27.7 in 128.  Heads of 32: 12 rows 14.6 in 16,
     * 14.7 in 32; 27 rows 17.2, 15.5, 16.1 in 64; 120 rows 23.3 in 64, 22.4 in 128.  8 sequences, 8 KV heads of 128: 12 rows 24.6 in
     * 16, 27.8 in 32; 28 rows 32.4, 29.7, 29.3 in 64; 112 rows 42.2 in 64, 41.3 in 128.
     * fp32 heads of 64 with steps for all blocks take 64 rows at least, whose two buffers hide the loads better (14 rows 26.7 in 16,
     * 23.2 in 64; 28 rows 29.6 in 32, 26.2; 7 rows of 1024 tokens 20.8, 16.5; but one sequence of 700 10.4, 10.6).  Other heads gain
     * with some 28 rows (32: 19.6, 18.2; 128: 49.6, 44.3) and lose with few (400 sequences of up to 4096 tokens, heads of 32: 107, 113;
     * 64 of 1024, heads of 128: 98, 110); the rule leaves them in the smallest. */
    k->wide = rows <= 16 ? 0 : rows <= 32 ? 1 : rows <= 64 ? 2 : 3;
    if (!half && a->HD == 64 && k->wide < 2 && units * imax(1, ceil_div(imin(a->max_kv, room), 128)) >= 512) k->wide = 2;
    const int tile = 16 << k->wide, step = k->wide < 2 ? 128 : k->wide == 3 && a->HD == 128 ? 32 : 64;
    /* (A grid ends below 2^32 threads, 2^24 blocks of 256: what has more row tiles takes several a block.) */
    k->MT = imin(ceil_div(rows, tile), (int)(((1 << 24) - 1) / ((units + 7) / 8 * 8)));
    const long long most = (long long)a->NKV * ((long long)a->c.R * G / tile + a->c.B) * imax(1, ceil_div(room, step));
    const long long tiles = units * k->MT, S = imax(1, ceil_div(imin(a->max_kv, room), step)), steps = tiles * S;
    const int slots = !half && a->HD == 128 && k->wide < 3 ? 256 : 512;
    /* A block a row tile: its steps (S) one after another, as often as the tiles fill the slots; dealt: an even share of all of them
     * (ragged ones: some 5/6) and of the tiles' beginnings, the line and the join, some 5 steps (fp32's of 128 keys are twice as
     * long).  Both in us, a tile a block first, 2 KV heads of 64: sequences of 500 fp16 tokens, 32 of them 9.1 and 10.6, 64 9.8 and
     * 13.9, 512 24 and 36; of 800, 64 13.2 and 14.5; of 1024, 64 15.5 and 14.8; of 2000, 512 64 and 71; of 4096, 400 113 and 99; trees
     * of 24 rows: 200 of 500 tokens 56 and 62, 256 of 3001 269 and 210.  2 KV heads of 32, fp16: 64 sequences of 500 9.2 and 12.1, of
     * 1024 14.3 and 12.5; 400 of 4096 103 and 88; fp32: 11.6 and 15.0 (dealt all the same), 17.5 and 15.3, 123 and 107.  8 KV heads of
     * 128, fp16: 16 of 500 13.0 and 17.6, of 1024 19.6 and 21.4 (dealt all the same), 64 of 1024 38 and 42; fp32: 31.5 and 31.2, 51 and
     * 42, 98 and 94. */
    const int still = 20 * ((tiles + slots - 1) / slots) * S <= 17 * tiles * (S + 2) / slots + (!half && step == 128 ? 50 : 100);
    /* (The join, a wave a row and head, has to fit a grid too.) */
    k->NB = still || most >= 1LL << 30 || a->c.R * a->NH > (1 << 26) - 4 ? 0 : steps < slots ? (int)steps : slots;
    /* A unit's beginning takes a block about as long as two steps (64 ragged fp16 requests, heads of 64, 26.5 us without, 24.0 with;
     * heads of 32 23.3, 20.9, fp32 29.3, 26.7; two long contexts, heads of 128, 78, 72; 8 sequences of 3000, heads of 128, 23.6, 23.4,
     * fp32 43.0, 43.4). */
    k->start = steps < slots ? 0 : 2;
}
static size_t tree_records(const tree_shape *k) { return (size_t)k->NB * 2 * (size_t)(16 << k->wide); }
static size_t tree_workspace(const sgpu_attn_tree_args *a, const tree_shape *k) {
    return k->NB ? tree_records(k) * ((size_t)a->HD + 2) * sizeof(float) + (size_t)a->c.R * (size_t)a->NH * 8 : 16;
}
size_t sgpu_attn_tree_workspace(const sgpu_attn_tree_args *a) {
    tree_shape k, h;
    if ((tree_check(a, 0) && tree_check(a, 1)) || a->c.R == 0 || a->c.B == 0) return 0;
    tree_plan(0, a, &k);
    tree_plan(1, a, &h);
    const size_t f32 = tree_workspace(a, &k), f16 = tree_workspace(a, &h);
    return f32 > f16 ? f32 : f16;
}
static int attn_tree(int half, const sgpu_attn_tree_args *a, void *ws, size_t ws_bytes, void *stream) {
    int rc = tree_check(a, half);
    if (rc || a->c.R == 0 || a->c.B == 0) return rc;
    const sgpu_paged_kv *c = &a->c;
    tree_shape p;
    tree_plan(half, a, &p);
    if (!ws || misaligned(ws, 16) || ws_bytes < tree_workspace(a, &p)) return SGPU_ERR_INVALID_ARG;
    tree_args k;
    memset(&k, 0, sizeof k);
    k.k = c->k; k.v = c->v; k.q = a->q; k.out = a->out; k.table = c->table; k.mask = a->mask;
    k.po = (float *)ws;
    k.pml = k.po + tree_records(&p) * (size_t)a->HD;
    k.desc = (int *)(k.pml + tree_records(&p) * 2);
    k.page_stride = c->page_stride; k.kv_row = c->kv_row; k.kv_head = c->kv_head; k.table_row = c->table_row;
    k.q_row = a->q_row; k.q_head = a->q_head; k.out_row = a->out_row; k.out_head = a->out_head; k.mask_row = a->mask_row;
    k.pages = c->pages; k.page = c->page; k.table_pages = c->pages ? c->table_pages : 0; k.NH = a->NH; k.scale = a->scale;
    k.MT = p.MT;
    for (k.shift = 0; 1LL << k.shift < c->page; k.shift++) {}      /* (any size, where the table has no entry) */
    if (1LL << k.shift != c->page) k.shift = -1;
    k.halves = c->page % 16 == 0 && c->kv_row <= 1 << 22;
    int B = c->B, R = c->R, NKV = a->NKV, NH = a->NH, G = NH / NKV, room = k.table_pages * k.page, rows = 16 << p.wide, n = R * NH;
    if (room == 0) {                              /* no keys, maybe no pages: a block's first loads, not used, read q's first row */
        k.k = k.v = a->q;
        k.kv_row = k.kv_head = 0;
        k.halves = 0;
    }
    int magic = G > 1 && (long long)R * G * G < 1LL << 32 ? (int)(unsigned)(((1ULL << 32) + (unsigned)G - 1) / (unsigned)G) : 0;
    const int j = a->HD == 32 ? 0 : a->HD == 64 ? 1 : 2;
    const int *q_start = c->q_start, *len = c->len;
    void *args[] = {&q_start, &len, &B, &R, &NKV, &G, &room, &p.NB, &p.start, &magic, &k};
    const unsigned blocks = p.NB ? (unsigned)p.NB : (unsigned)(ceil_div((long long)B * NKV, 8) * 8 * p.MT);
    rc = sgpu_internal_paged_launch(SGPU_PG_TREE + 3 * (4 * half + p.wide) + j, blocks, 256, args, stream);
    if (rc || !p.NB) return rc;
    void *jargs[] = {&k.desc, &k.po, &k.pml, &k.out, &k.out_row, &k.out_head, &NH, &n, &rows};
    return sgpu_internal_paged_launch(SGPU_PG_TREE + 24 + j, (unsigned)ceil_div(n, 4), 256, jargs, stream);
}
int sgpu_attn_tree(const sgpu_attn_tree_args *a, void *ws, size_t ws_bytes, void *stream) {
    return attn_tree(0, a, ws, ws_bytes, stream);
}
int sgpu_attn_tree_h(const sgpu_attn_tree_args *a, void *ws, size_t ws_bytes, void *stream) {
    return attn_tree(1, a, ws, ws_bytes, stream);
}

/* ---- logits ---- */
/* paged_logits of sgpu_paged.hip */
typedef struct {
    const void *x;
    void *y;
    const int *tok, *span, *bias_id, *bias_span;
    const float *rep, *freq, *pres, *bias;
    const uint32_t *allow;
    long long x_row, y_row, allow_row;
    int rows, V, n_tok, n_bias, C, groups;
} logits_args;

#define LOGITS_ROWS (1 << 21)                     /* the most rows of a launch (one block a row from 512 rows on) */
static int logits_adjust(int half, const sgpu_logits_args *p, void *stream) {
    if (!p || p->rows < 0 || p->rows >= 1 << 24 || p->V < 1 || p->V > 1 << 30 || p->n_tok < 0 || p->n_bias < 0)
        return SGPU_ERR_INVALID_ARG;
    if (p->rows == 0) return SGPU_OK;
    const size_t size = half ? 2 : 4;
    const long long C = ceil_div(p->V, 8192);
    if (!p->x || !p->y || misaligned(p->x, size) || misaligned(p->y, size) || p->x_row < p->V || p->y_row < p->V ||
        (p->x == p->y && p->x_row != p->y_row) || p->rows * C >= 1LL << 31)
        return SGPU_ERR_INVALID_ARG;
    if (p->span && ((p->n_tok > 0 && !p->tok) || misaligned(p->span, 4) || misaligned(p->tok, 4))) return SGPU_ERR_INVALID_ARG;
    if (misaligned(p->rep, 4) || misaligned(p->freq, 4) || misaligned(p->pres, 4)) return SGPU_ERR_INVALID_ARG;
    const int bias = p->bias_span && p->n_bias > 0;
    if (bias && (!p->bias_id || !p->bias || misaligned(p->bias_span, 4) || misaligned(p->bias_id, 4) || misaligned(p->bias, 4)))
        return SGPU_ERR_INVALID_ARG;
    if (p->allow && (misaligned(p->allow, 4) || (p->allow_row != 0 && p->allow_row < ceil_div(p->V, 32)))) return SGPU_ERR_INVALID_ARG;
    logits_args a = {p->x, p->y, p->tok, p->span, p->bias_id, p->bias_span, p->rep, p->freq, p->pres, p->bias, p->allow,
                     p->x_row, p->y_row, p->allow_row, p->rows, p->V, p->n_tok, p->n_bias, (int)C, 0};
    a.groups = imin((int)C, imax(1, 512 / p->rows));          /* blocks of a row: two a CU in all (figures at the kernel) */
    a.groups = ceil_div(C, ceil_div(C, a.groups));
    /* A grid ends below 2^32 threads, 2^22 blocks here: more rows in parts. */
    for (long long r0 = 0; r0 < p->rows; r0 += LOGITS_ROWS) {
        logits_args part = a;
        part.rows = imin(p->rows - (int)r0, LOGITS_ROWS);
        part.x = (const char *)a.x + r0 * a.x_row * (long long)size;
        part.y = (char *)a.y + r0 * a.y_row * (long long)size;
        if (a.span) part.span = a.span + 4 * r0;
        if (a.rep) part.rep = a.rep + r0;
        if (a.freq) part.freq = a.freq + r0;
        if (a.pres) part.pres = a.pres + r0;
        if (a.bias_span) part.bias_span = a.bias_span + 2 * r0;
        if (a.allow) part.allow = a.allow + r0 * a.allow_row;
        void *args[] = {&part};
        int rc = sgpu_internal_paged_launch(SGPU_PG_LOGITS + 2 * bias + half, (unsigned)(part.rows * a.groups), 1024, args, stream);
        if (rc) return rc;
    }
    return SGPU_OK;
}
int sgpu_logits_adjust(const sgpu_logits_args *a, void *stream) { return logits_adjust(0, a, stream); }
int sgpu_logits_adjust_h(const sgpu_logits_args *a, void *stream) { return logits_adjust(1, a, stream); }
