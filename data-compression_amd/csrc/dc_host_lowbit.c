/*
 * dc_host_lowbit.c -- entry points of the fixed-rate operators (include/dc_gpu.h): the key/value cache in 4 or 8 bits
 * (dc_kv.hip) and the 8-bit activation checkpoints (dc_act.hip).  Checks of arguments, the choice of a kernel's variant
 * and the launch; no state but the sticky status word (and the calling thread's error message), so that calls on several
 * streams and from several threads do not meet.
 */
#define __HIP_PLATFORM_AMD__ 1
#include <hip/hip_runtime_api.h>
#include <pthread.h>
#include <stdint.h>
#include <string.h>

#include "dc_shared.h"
#include "../../include/dc_gpu.h"

int dc_set_error(int code, const char* msg);
unsigned* dc_kv_status_word(void);

#define REFUSE(msg) return dc_set_error(DC_ERR_ARG, msg)

/* a launch has fewer than 2^32 threads, here in workgroups of 256 */
enum { MOST_GROUPS = (1 << 24) - 1 };
#define MOST_ACT (2048ll * MOST_GROUPS)

/* the high half of n times this is n / d where n d < 2^64 (2^64 / d, rounded up); 0 stands for d = 1 */
static unsigned long long inverse(unsigned long long d) { return d <= 1 ? 0 : ~0ull / d + 1; }

/* the library is started and the stream is one of its device; HIP's default stream belongs to whichever is the current one */
static int ready(void* stream) {
    const int rc = dc_init(0);
    if (rc) return rc;
    int device = 0;                                             /* (hipGetDevice is the shorter call) */
    if ((stream ? hipStreamGetDevice((hipStream_t)stream, &device) : hipGetDevice(&device)) != hipSuccess)
        (void)hipGetLastError();                                /* (the launch will say) */
    else if (device != dc_get_device())
        REFUSE("the stream (the default stream: the current device) is not of the library's device");
    return DC_OK;
}

static int size_of(int dtype) { return dtype == DC_F32 ? 4 : dtype == DC_F16 || dtype == DC_BF16 ? 2 : 0; }

size_t dc_kv_page_bytes(int page_size, int heads, int head_dim, int bits) {
    if (page_size < 16 || page_size % 16 || page_size > (1 << 30) || heads < 1 || heads > (1 << 20) || head_dim < 32 ||
        head_dim > 256 || head_dim % 32 || (bits != 4 && bits != 8))
        return 0;
    return (size_t)page_size * (size_t)heads * (size_t)(2 * (head_dim * bits / 8) + 8);
}

/* the checks and the fields that the three cache operators share; rows of `heads` heads */
static int common(const dc_kv_cache* c, const dc_kv_batch* at, KvArgs* a) {
    if (!c || !at) REFUSE("cache: no cache or no positions");
    const size_t page = dc_kv_page_bytes(c->page_size, c->heads, c->head_dim, c->bits);
    if (!page)
        REFUSE("cache: page_size is a multiple of 16, head_dim a multiple of 32 up to 256, bits 4 or 8, heads at least 1");
    if (c->pages < 1 || !c->data || ((uintptr_t)c->data & 15u)) REFUSE("cache: data is 16-byte aligned, pages at least 1");
    if (c->pages > (long long)((1ull << 62) / page)) REFUSE("cache: too many pages");
    if (at->batch < 0 || at->tokens < 0) REFUSE("cache: batch and tokens are not negative");
    if (at->batch && at->tokens && !at->start) REFUSE("cache: start is missing");
    if (at->table && (at->table_width < 1 || at->table_stride < at->table_width))
        REFUSE("cache: table_width is at least 1, table_stride at least table_width");
    if (!at->table && at->batch > c->pages) REFUSE("cache: without a table each sequence has a page");
    memset(a, 0, sizeof *a);
    a->data = (uint8_t*)c->data;
    a->pages = c->pages;
    a->head_bytes = (long long)(page / (size_t)c->heads);
    a->page = c->page_size;
    a->heads = c->heads;
    a->dim = c->head_dim;
    a->bits = c->bits;
    a->batch = at->batch;
    a->tokens = at->tokens;
    a->start = at->start;
    a->lens = at->lens;
    a->table = at->table;
    a->zero_padding = at->zero_padding != 0;
    a->table_stride = at->table_stride;
    a->capacity = (long long)c->page_size * (at->table ? at->table_width : 1);
    if (a->capacity > (1ll << 30)) a->capacity = 1ll << 30;      /* positions are 32-bit */
    a->page_inv = inverse((unsigned long long)c->page_size);
    a->blocks_inv = inverse((unsigned long long)c->page_size / 16);
    a->heads_inv = inverse((unsigned long long)c->heads);
    return DC_OK;
}

static unsigned low_bit(unsigned x) { return x & (0u - x); }

/* whether rows at p with these strides may be accessed in pieces of `bytes` */
static int fits(const void* p, const long long* s, int size, unsigned bytes) {
    const uintptr_t m = bytes - 1;
    if ((uintptr_t)p & m) return 0;
    for (int i = 0; i < 3; i++)
        if ((uintptr_t)s[i] * (uintptr_t)size & m) return 0;
    return 1;
}

static int rows_call(const dc_kv_cache* c, const dc_kv_batch* at, int dtype, const void* k, const long long* ks,
                     const void* v, const long long* vs, void* stream, int write) {
    KvArgs a;
    int rc = common(c, at, &a);
    if (rc) return rc;
    const int size = size_of(dtype);
    if (!size) REFUSE("cache: dtype is DC_F32, DC_F16 or DC_BF16");
    if (at->batch == 0 || at->tokens == 0) return DC_OK;
    if (!k || !v || !ks || !vs) REFUSE("cache: keys, values and their strides are needed");
    if (((uintptr_t)k | (uintptr_t)v) & (uintptr_t)(size - 1)) REFUSE("cache: keys and values are aligned to their type");
    if ((long long)at->batch * at->tokens > (1ll << 30) / c->heads) REFUSE("cache: too many rows in one call");
    a.blocks = (int)(((long long)at->tokens + 30) / 16);        /* at any place within the first block */
    a.tokens_inv = inverse((unsigned long long)a.blocks);
    a.rows = (long long)at->batch * a.blocks * c->heads * (write ? 2 : 1);
    if ((a.rows + 3) / 4 > MOST_GROUPS) REFUSE("cache: too many rows in one call");
    a.k = k;
    a.v = v;
    memcpy(a.ks, ks, sizeof a.ks);
    memcpy(a.vs, vs, sizeof a.vs);
    a.dtype = dtype;
    /* floats that no cache holds pass them (4 sequences of 16384 read, bf16: 62 us, so 47; 16 of 4095 written, f16, and read
       back: 112, so 103); fewer do not (3 of 4095, f16, read: 12.1 us, so 12.8, written: 17.0, so 18.0), and what uses them next
       finds them there */
    a.past = 2.0 * at->batch * at->tokens * c->heads * c->head_dim * size > 128e6;
    const unsigned piece = low_bit((unsigned)(c->head_dim / 16 * size));
    a.vec = fits(k, ks, size, piece > 16 ? 16 : piece) && fits(v, vs, size, piece > 16 ? 16 : piece);
    if ((rc = ready(stream))) return rc;
    a.status = dc_kv_status_word();
    return dc_launch_kv_rows(&a, write, (dc_hip_stream)stream) ? dc_set_error(DC_ERR_HIP, "cache: the launch failed") : DC_OK;
}

int dc_kv_write_device(const dc_kv_cache* cache, const dc_kv_batch* at, int dtype, const void* d_k,
                       const long long* k_strides, const void* d_v, const long long* v_strides, void* stream) {
    return rows_call(cache, at, dtype, d_k, k_strides, d_v, v_strides, stream, 1);
}

int dc_kv_read_device(const dc_kv_cache* cache, const dc_kv_batch* at, int dtype, void* d_k, const long long* k_strides,
                      void* d_v, const long long* v_strides, void* stream) {
    return rows_call(cache, at, dtype, d_k, k_strides, d_v, v_strides, stream, 0);
}

/* How the attention is cut.  Query rows (tokens x the group that shares a head) in tiles of 16, or of as many as a wave's
 * registers hold where there are more.  The cache's positions in up to `splits` pieces a sequence, so that there are
 * about 768 workgroups, 3 per compute unit (with the join, 48 sequences of up to 8192 positions, 8 heads: 512 84 us, 768 76,
 * 1024 75, 2048 76; 20 of them: 38, 38, 40, 48), or half of that where a compute unit holds two of them, wide tiles and long
 * rows (16 sequences of 8192, heads of 256: 256 37 us, 384 32, 768 38; 8 queries each, heads of 64: 256 31, 384 27, 768
 * 33); up to twice the even number of pieces, for sequences longer than the others.  At most 256 pieces, as the join takes a
 * thread for each: one sequence of 1 or 2 heads then has 256 or 512 workgroups, whatever the aim (262143 positions, 2 heads:
 * 21 us).
 * None up to 640 positions: there a second kernel, which joins the pieces, costs what they save (8 heads, 517 positions:
 * 9.6 us in one piece, 7.0 + 2.8 in three). */
static int plan(const dc_kv_cache* c, int batch, int tokens, int q_heads, long long max_context, KvArgs* a) {
    if (q_heads < 1 || q_heads % c->heads) return 1;
    const long long group = q_heads / c->heads, rows = (long long)tokens * group;
    if (rows > (1ll << 30)) return 1;
    a->group = (int)group;
    a->group_inv = inverse((unsigned long long)group);
    a->cols = rows <= 16 ? 16 : (unsigned)dc_kv_wide_cols(c->head_dim);
    a->tiles = (unsigned)((rows + a->cols - 1) / a->cols);
    a->row_slots = (unsigned)rows;
    const long long base = (long long)batch * c->heads * a->tiles;
    if (base > (1ll << 30)) return 1;
    if (max_context > 1ll << 30) max_context = 1ll << 30;       /* (positions are 32-bit) */
    const int AIM = a->cols == 16 && c->head_dim <= 128 ? 768 : 384;
    enum { SHORT = 640, LEAST = 256, MOST = 256 };
    long long splits = 1;
    if (base > 0 && base < AIM && max_context > SHORT) {
        const long long most = (max_context + LEAST - 1) / LEAST;
        splits = 2 * ((AIM + base - 1) / base);
        if (splits > most) splits = most;
        if (splits > MOST) splits = MOST;
    }
    a->splits = (unsigned)splits;
    a->target = base < AIM ? (unsigned)(AIM - base / 2) : 1u;
    return 0;
}

static size_t workspace_of(const KvArgs* a, int batch) {
    if (a->splits <= 1) return 0;
    return (size_t)batch * (size_t)a->heads * a->row_slots * a->splits * ((size_t)a->dim + 2) * sizeof(float);
}

size_t dc_kv_attention_workspace(const dc_kv_cache* cache, int batch, int tokens, int q_heads, long long max_context) {
    KvArgs a;
    if (!cache || batch < 1 || tokens < 1 || max_context < 0 ||
        !dc_kv_page_bytes(cache->page_size, cache->heads, cache->head_dim, cache->bits))
        return 0;
    memset(&a, 0, sizeof a);
    a.heads = cache->heads;
    a.dim = cache->head_dim;
    return plan(cache, batch, tokens, q_heads, max_context, &a) ? 0 : workspace_of(&a, batch);
}

int dc_kv_attention_device(const dc_kv_cache* cache, const dc_kv_batch* at, int dtype, int q_heads, const void* d_q,
                           const long long* q_strides, float scale, int causal, long long max_context, void* d_out,
                           const long long* out_strides, float* d_lse, void* d_workspace, size_t workspace_bytes,
                           void* stream) {
    KvArgs a;
    int rc = common(cache, at, &a);
    if (rc) return rc;
    if (dtype != DC_F16 && dtype != DC_BF16) REFUSE("attention: queries are DC_F16 or DC_BF16");
    if (max_context < 0) REFUSE("attention: max_context is not negative");
    if (q_heads < 1 || q_heads % cache->heads) REFUSE("attention: q_heads is a multiple of the cache's heads");
    if (at->batch == 0 || at->tokens == 0) return DC_OK;
    if (!d_q || !d_out || !q_strides || !out_strides) REFUSE("attention: queries, output and their strides are needed");
    if (((uintptr_t)d_q | (uintptr_t)d_out) & 1u || (uintptr_t)d_lse & 3u)
        REFUSE("attention: queries, output and lse are aligned to their types");
    if (plan(cache, at->batch, at->tokens, q_heads, max_context, &a)) REFUSE("attention: too many query rows in one call");
    if ((long long)a.splits * a.tiles * a.heads * a.batch > MOST_GROUPS ||
        (a.splits > 1 && (long long)a.row_slots * a.heads * a.batch * 8 > MOST_GROUPS))
        REFUSE("attention: too many query rows in one call");
    const size_t need = workspace_of(&a, at->batch);
    if (need && (!d_workspace || workspace_bytes < need || ((uintptr_t)d_workspace & 15u)))
        REFUSE("attention: the workspace is missing, too small or not 16-byte aligned (dc_kv_attention_workspace)");
    a.k = d_q;
    a.v = d_out;
    memcpy(a.ks, q_strides, sizeof a.ks);
    memcpy(a.vs, out_strides, sizeof a.vs);
    a.dtype = dtype;
    /* codes that no cache holds until the next call are read past them (100 sequences of up to 4096, 0.36 GB: 80 us, so 76;
       16 of 16384, 0.29 GB: 58, so 53; 2 of 65536, 0.14 GB: 34, so 37) */
    const long long longest = max_context < a.capacity ? max_context : a.capacity;
    a.past = 1.0 * at->batch * longest * a.head_bytes / a.page * a.heads > 256e6;
    /* outputs are stored by units of head_dim / 16 values, and by the join of few pieces four values at once */
    unsigned piece = low_bit((unsigned)(cache->head_dim / 16 * 2));
    if (piece > 16) piece = 16;
    if (piece < 8 && a.splits > 1 && a.splits <= DC_KV_JOIN_FEW) piece = 8;
    a.vec = fits(d_q, q_strides, 2, 16);
    a.vec_out = fits(d_out, out_strides, 2, piece);
    a.causal = causal != 0;
    a.scale = scale;
    a.lse = d_lse;
    a.part = (float*)d_workspace;
    a.part_ml = need ? a.part + (size_t)at->batch * (size_t)a.heads * a.row_slots * a.splits * (size_t)a.dim : NULL;
    if ((rc = ready(stream))) return rc;
    a.status = dc_kv_status_word();
    return dc_launch_kv_attention(&a, (dc_hip_stream)stream) ? dc_set_error(DC_ERR_HIP, "attention: the launch failed") : DC_OK;
}

int dc_kv_status(void* stream, unsigned* status_out, int reset) {
    if (!status_out) REFUSE("status: nowhere to put it");
    int rc = ready(stream);
    if (rc) return rc;
    hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
    const int unsure = hipStreamIsCapturing((hipStream_t)stream, &cap) != hipSuccess;   /* (the default stream beside a capture) */
    if (unsure) (void)hipGetLastError();                        /* (not for the next launch to find) */
    if (unsure || cap != hipStreamCaptureStatusNone) REFUSE("status: the stream is being captured");
    /* a reset takes the word and clears it in one step, into the word beside it: a bit that another stream's call sets
     * meanwhile is in this answer or in the next (the lock is for that place) */
    static pthread_mutex_t lock = PTHREAD_MUTEX_INITIALIZER;
    unsigned* w = dc_kv_status_word();
    if (reset) pthread_mutex_lock(&lock);
    const int bad = (reset && dc_launch_kv_take(w, (dc_hip_stream)stream)) ||
                    hipMemcpyAsync(status_out, w + (reset != 0), 4, hipMemcpyDeviceToHost, (hipStream_t)stream) != hipSuccess ||
                    hipStreamSynchronize((hipStream_t)stream) != hipSuccess;
    if (reset) pthread_mutex_unlock(&lock);
    return bad ? dc_set_error(DC_ERR_HIP, "status: the read failed") : DC_OK;
}

/* ---- activation checkpoints ------------------------------------------------------------------------------ */
size_t dc_act_bytes(long long n) { return n < 0 || n > MOST_ACT ? 0 : (size_t)((n + 31) / 32) * 33u; }

/* one array of the call: 0 flat and aligned, 1 rows apart in whole 8s and aligned, 2 neither */
static int shape_of(const void* p, long long ld, long long rows, long long cols, int size) {
    if (!p) return 0;
    const int aligned = ((uintptr_t)p & 15u) == 0;
    if (aligned && (ld == cols || rows == 1)) return 0;
    return aligned && cols % 8 == 0 && (uintptr_t)ld * (uintptr_t)size % 16 == 0 ? 1 : 2;
}

static int act_call(ActArgs* a, int back, void* stream) {
    const int size = size_of(a->dtype);
    if (!size) REFUSE("activation: dtype is DC_F32, DC_F16 or DC_BF16");
    if (a->kind != DC_ACT_NONE && a->kind != DC_ACT_SILU && a->kind != DC_ACT_GELU) REFUSE("activation: unknown kind");
    if (a->rows < 0 || a->cols < 0 || (a->cols && a->rows > MOST_ACT / a->cols)) REFUSE("activation: at most 2^35 - 2048 values");
    if (a->rows == 0 || a->cols == 0) return DC_OK;
    const int works = a->kind != DC_ACT_NONE;
    if (!a->kept || (a->gated && !a->kept_up)) REFUSE("activation: a checkpoint is missing");
    if (((uintptr_t)a->kept | (uintptr_t)a->kept_up) & 15u) REFUSE("activation: checkpoints are 16-byte aligned");
    if (back ? !a->dx || (works != !!a->x) || (!works && a->y) : !a->x || (works != !!a->y))
        REFUSE("activation: an array is missing, or is not used by this kind");
    if (!works && (a->gated || a->dup)) REFUSE("activation: a checkpoint alone has one input");
    const void* arrays[5] = {a->x, a->up, a->y, a->dx, a->dup};
    const long long lds[5] = {a->ldx, a->ldup, a->ldy, a->lddx, a->lddup};
    int mode = 0, apart = 0;
    for (int i = 0; i < 5; i++) {
        if (!arrays[i]) continue;
        if (lds[i] < a->cols) REFUSE("activation: rows are at least cols apart");
        if ((uintptr_t)arrays[i] & (uintptr_t)(size - 1)) REFUSE("activation: arrays are aligned to their type");
        const int s = shape_of(arrays[i], lds[i], a->rows, a->cols, size);
        if (s == 2) mode = 2;
        if (s == 1) apart = 1;
    }
    /* with one array's rows apart all are taken row by row: then rows of 8s everywhere */
    if (mode == 0 && apart) {
        mode = 1;
        for (int i = 0; i < 5; i++)
            if (arrays[i] && (a->cols % 8 || (a->rows > 1 && (uintptr_t)lds[i] * (uintptr_t)size % 16))) mode = 2;
    }
    a->mode = mode;
    a->n = a->rows * a->cols;
    /* outputs that no cache holds are written past them (134M bf16 values forward 113 us, so 101, loaded 73 and 67, a
       gated backward of 67M 118 and 113) */
    a->past = (double)a->n * size * (!!a->y + !!a->dx + !!a->dup) > 128e6;
    a->groups = (a->n + 31) / 32;
    a->cols8_inv = inverse((unsigned long long)(a->cols / 8));
    const int rc = ready(stream);
    if (rc) return rc;
    return dc_launch_act(a, back, (dc_hip_stream)stream) ? dc_set_error(DC_ERR_HIP, "activation: the launch failed") : DC_OK;
}

int dc_act_forward_device(int kind, int dtype, long long rows, long long cols, const void* d_x, long long ldx,
                          const void* d_up, long long ldup, void* d_y, long long ldy, void* d_kept, void* d_kept_up,
                          void* stream) {
    ActArgs a;
    memset(&a, 0, sizeof a);
    a.kind = kind;
    a.gated = d_up != NULL;
    a.dtype = dtype;
    a.rows = rows;
    a.cols = cols;
    a.x = d_x;
    a.ldx = ldx;
    a.up = d_up;
    a.ldup = ldup;
    a.y = d_y;
    a.ldy = ldy;
    a.kept = (uint8_t*)d_kept;
    a.kept_up = (uint8_t*)d_kept_up;
    return act_call(&a, 0, stream);
}

int dc_act_backward_device(int kind, int dtype, long long rows, long long cols, const void* d_dy, long long lddy,
                           const void* d_kept, const void* d_kept_up, void* d_dx, long long lddx, void* d_dup,
                           long long lddup, void* d_y, long long ldy, void* stream) {
    if (!d_kept_up != !d_dup) REFUSE("activation: kept_up and dup belong together");
    ActArgs a;
    memset(&a, 0, sizeof a);
    a.kind = kind;
    a.gated = d_dup != NULL;
    a.dtype = dtype;
    a.rows = rows;
    a.cols = cols;
    a.x = d_dy;
    a.ldx = lddy;
    a.dx = d_dx;
    a.lddx = lddx;
    a.dup = d_dup;
    a.lddup = lddup;
    a.y = d_y;
    a.ldy = ldy;
    a.kept = (uint8_t*)d_kept;
    a.kept_up = (uint8_t*)d_kept_up;
    return act_call(&a, 1, stream);
}
