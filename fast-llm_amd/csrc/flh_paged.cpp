// flh_paged.cpp -- entry points of the paged key/value cache, the rotary
// positions and the attention (include/fastllm_hip.h): argument checks, then
// one call of the launchers.  Nothing is launched on an error.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include <new>
#include <vector>
#include "../../include/fastllm_hip.h"
#include "flh_internal.h"
#include "flh_status.h"

using namespace flh;

struct flh_rope_table {
    RopePair * dev;
    uint32_t n_rot, first, halves;
};

namespace {

bool off(const void * p, uintptr_t align) { return ((uintptr_t)p & (align - 1)) != 0; }
bool pow2_page(uint32_t n) { return n >= 1 && n <= 65536 && (n & (n - 1)) == 0; }
uintptr_t elem(uint32_t dtype) { return dtype == FLH_DT_F32 ? 4 : 2; }

}  // namespace

int flh::check_kv_cache(const flh_kv_cache * c) {
    if (!c) return set_error(FLH_ERR_ARG, "kv cache: null");
    if (c->dtype != FLH_DT_F16 && c->dtype != FLH_DT_BF16)
        return set_error(FLH_ERR_UNSUPPORTED, "kv cache: dtype must be F16 or BF16");
    if (!c->k || !c->v || off(c->k, 16) || off(c->v, 16))
        return set_error(FLH_ERR_ARG, "kv cache: k and v must be non-null and 16-byte aligned");
    if (!pow2_page(c->page_size)) return set_error(FLH_ERR_UNSUPPORTED, "kv cache: page_size must be a power of two up to 65536");
    if (c->n_pages == 0 || (uint64_t)c->n_pages * c->page_size >= 0xFFFFFFFFull)
        return set_error(FLH_ERR_ARG, "kv cache: n_pages * page_size must be in 1 .. 2^32 - 2");
    if (c->n_kv_head == 0 || c->n_kv_head > 65535) return set_error(FLH_ERR_ARG, "kv cache: n_kv_head must be in 1 .. 65535");
    if (c->d_k == 0 || c->d_k > 256 || c->d_k % 8 || c->d_v == 0 || c->d_v > 256 || c->d_v % 8)
        return set_error(FLH_ERR_UNSUPPORTED, "kv cache: d_k and d_v must be multiples of 8 up to 256");
    if ((c->k_page | c->k_tok | c->k_head | c->v_page | c->v_tok | c->v_head) & 7)
        return set_error(FLH_ERR_ARG, "kv cache: strides must be multiples of 8 elements");
    if ((c->k_page | c->k_tok | c->v_page | c->v_tok) >= (1ull << 31) || (c->k_head | c->v_head) >= (1ull << 40))
        return set_error(FLH_ERR_UNSUPPORTED, "kv cache: page and token strides must be below 2^31 elements, head strides below 2^40");
    return FLH_OK;
}

namespace {

// [tok][head][d] elements at these strides
struct Rows {
    const void * p;
    uint64_t tok, head;
    uint32_t d;
};
typedef unsigned __int128 u128;
// Whether two sets of n_tok x n_head rows (of el bytes an element, both counts > 0) share a
// byte.  Their extents tell, or, where both take equal steps, the places within a
// step: columns of the same rows, or heads that stand in turn, are apart.  Else: yes.
bool overlap(const Rows & a, const Rows & b, uint32_t n_tok, uint32_t n_head, uintptr_t el) {
    const u128 pa = (uintptr_t)a.p, pb = (uintptr_t)b.p;
    auto row = [&](const Rows & r) { return ((u128)(n_head - 1) * r.head + r.d) * el; };
    auto all = [&](const Rows & r) { return (u128)(n_tok - 1) * r.tok * el + row(r); };
    if (pa + all(a) <= pb || pb + all(b) <= pa) return false;
    // pieces of na and nb bytes, each a multiple of `step` bytes behind the first
    auto apart = [&](u128 step, u128 na, u128 nb) {
        if (step == 0 || na > step || nb > step) return false;
        const u128 at = pb >= pa ? (pb - pa) % step : (step - (pa - pb) % step) % step;
        return at >= na && at + nb <= step;
    };
    if (a.tok == b.tok && apart((u128)a.tok * el, row(a), row(b))) return false;
    if (a.head == b.head && a.head && (n_tok == 1 || (a.tok % a.head == 0 && b.tok % b.head == 0)) &&
        apart((u128)a.head * el, a.d * el, b.d * el)) return false;
    return true;
}

int check_rope(const flh_rope_table * r, uint32_t d, const int32_t * pos) {
    if (!r) return FLH_OK;
    if (r->first + r->n_rot > d) return set_error(FLH_ERR_ARG, "rope: first + n_rot exceeds the head");
    if (!pos || off(pos, 4)) return set_error(FLH_ERR_ARG, "rope: pos must be non-null and 4-byte aligned");
    return FLH_OK;
}
int check_turned(const void * x, uint64_t x_tok, uint64_t x_head, const void * y, uint64_t y_tok, uint64_t y_head,
                 uint32_t n_tok, uint32_t n_head, uint32_t d, uint32_t dtype) {
    const uintptr_t el = elem(dtype);
    if (!x || !y || off(x, el) || off(y, el)) return set_error(FLH_ERR_ARG, "rope: x and y must be non-null and element aligned");
    if (x == y && x_tok == y_tok && x_head == y_head) return FLH_OK;
    if (overlap({x, x_tok, x_head, d}, {y, y_tok, y_head, d}, n_tok, n_head, el))
        return set_error(FLH_ERR_ARG, "rope: y overlaps x with other strides or another address");
    return FLH_OK;
}
void set_rope(RopeArgs & a, const flh_rope_table * r) {
    a.rot = r ? r->dev : nullptr;
    a.n_rot = r ? r->n_rot : 0;
    a.first = r ? r->first : 0;
    a.halves = r ? r->halves : 0;
}

int attn_args(const flh_kv_cache * c, const flh_attn_p * p, AttnTreeArgs & a) {
    if (int rc = check_kv_cache(c)) return rc;
    if (!p) return set_error(FLH_ERR_ARG, "attention: null arguments");
    if (p->dtype > FLH_DT_BF16) return set_error(FLH_ERR_ARG, "attention: unknown dtype");
    if (p->dtype != FLH_DT_F32 && p->dtype != c->dtype)
        return set_error(FLH_ERR_UNSUPPORTED, "attention: q must be F32 or of the cache's dtype");
    if (p->n_head == 0 || p->n_head % c->n_kv_head) return set_error(FLH_ERR_ARG, "attention: n_head must be a multiple of n_kv_head");
    const uint32_t group = p->n_head / c->n_kv_head;
    if ((uint64_t)p->n_tok * group >= (1ull << 30)) return set_error(FLH_ERR_UNSUPPORTED, "attention: n_tok * (n_head / n_kv_head) must be below 2^30");
    if (!(p->scale >= 0.f) || !isfinite(p->scale)) return set_error(FLH_ERR_ARG, "attention: scale must be finite and >= 0");
    if (p->window && !p->causal) return set_error(FLH_ERR_ARG, "attention: a window needs causal");
    const uint64_t keys = (uint64_t)p->table_stride * c->page_size;
    if (keys > (1ull << 30)) return set_error(FLH_ERR_UNSUPPORTED, "attention: table_stride * page_size must be at most 2^30");
    // units of work are counted in 32 bits (strips of 16 rows or more, tiles of 64 keys or more and ATTN_ITEM units a strip)
    if ((double)c->n_kv_head * ((double)p->n_tok * group / 16 + 2.0 * p->n_seq) * ((double)keys / 64 + 1 + ATTN_ITEM) >= 4.0e9)
        return set_error(FLH_ERR_UNSUPPORTED, "attention: too much work for one call (rows times table length)");
    a = AttnTreeArgs{};
    a.q = p->q; a.out = p->out; a.q_start = p->q_start; a.kv_len = p->kv_len; a.table = p->table; a.ws = p->ws;
    a.k = c->k; a.v = c->v;
    a.q_tok = p->q_tok; a.q_head = p->q_head; a.o_tok = p->o_tok; a.o_head = p->o_head;
    a.k_page = (uint32_t)(2 * c->k_page); a.k_tok = (uint32_t)(2 * c->k_tok); a.k_head = 2 * c->k_head;
    a.v_page = (uint32_t)(2 * c->v_page); a.v_tok = (uint32_t)(2 * c->v_tok); a.v_head = 2 * c->v_head;
    a.n_pages = c->n_pages; a.sh = (uint32_t)__builtin_ctz(c->page_size); a.n_kv = c->n_kv_head;
    a.dk = c->d_k; a.dv = c->d_v; a.group = group;
    a.n_seq = p->n_seq; a.n_tok = p->n_tok; a.max_q = p->max_q; a.table_stride = p->table_stride;
    a.causal = p->causal != 0; a.window = p->window; a.pmask = c->page_size - 1; a.scale = p->scale;
    return FLH_OK;
}

// the rest of a call: pointers, workspace, launches
int attn_run(const flh_kv_cache * c, const flh_attn_p * p, const AttnTreeArgs & a, void * stream) {
    if (p->n_tok && p->n_seq) {
        const uintptr_t el = elem(p->dtype);
        if (!p->q || !p->out || off(p->q, el) || off(p->out, el))
            return set_error(FLH_ERR_ARG, "attention: q and out must be non-null and element aligned");
        if (!p->q_start || !p->kv_len || off(p->q_start, 4) || off(p->kv_len, 4) || off(p->table, 4) || (!p->table && p->table_stride))
            return set_error(FLH_ERR_ARG, "attention: q_start, kv_len and table must be non-null and 4-byte aligned");
        if (overlap({p->q, p->q_tok, p->q_head, c->d_k}, {p->out, p->o_tok, p->o_head, c->d_v}, p->n_tok, p->n_head, el))
            return set_error(FLH_ERR_ARG, "attention: out overlaps q");
        const size_t need = attn_ws_bytes(a, p->dtype);
        if (need && (!p->ws || off(p->ws, 16) || p->ws_bytes < need))
            return set_error(FLH_ERR_ARG, a.tree_stride ? "attention: ws must be 16-byte aligned and of flh_tree_attn_ws_bytes"
                                                        : "attention: ws must be 16-byte aligned and of flh_paged_attn_ws_bytes");
    }
    if (int rc = need_device()) return rc;
    if (p->n_tok == 0 || p->n_seq == 0) return FLH_OK;
    // two launches that belong together: another thread's call in between would take the
    // workspace, which calls on one stream may share
    const StreamTurn turn(stream, true);
    return launch_attn(a, p->dtype, c->dtype, (hipStream_t)stream);
}

}  // namespace

extern "C" {

int flh_kv_plan(const flh_kv_plan_p * p, void * stream) {
    if (!p) return set_error(FLH_ERR_ARG, "kv plan: null arguments");
    if (!pow2_page(p->page_size)) return set_error(FLH_ERR_UNSUPPORTED, "kv plan: page_size must be a power of two up to 65536");
    if (!p->taken || !p->q_start || (p->n_seq && (!p->held || !p->add || !p->kv_len || !p->table || p->table_stride == 0)) ||
        (p->n_free && !p->free_pages) || (p->max_tok && !p->slot))
        return set_error(FLH_ERR_ARG, "kv plan: null argument");
    if ((uint64_t)p->table_stride * p->page_size > (1ull << 31))
        return set_error(FLH_ERR_UNSUPPORTED, "kv plan: table_stride * page_size must be at most 2^31");
    if (p->max_tok > (1u << 31)) return set_error(FLH_ERR_UNSUPPORTED, "kv plan: max_tok must be at most 2^31");
    for (const void * q : {(const void *)p->held, (const void *)p->add, (const void *)p->free_pages, (const void *)p->taken_in,
                           (const void *)p->taken, (const void *)p->table, (const void *)p->q_start, (const void *)p->kv_len,
                           (const void *)p->slot, (const void *)p->pos, (const void *)p->info})
        if (off(q, 4)) return set_error(FLH_ERR_ARG, "kv plan: arrays must be 4-byte aligned");
    if (int rc = need_device()) return rc;
    const StreamTurn turn(stream, true);                          // (two launches, as below)
    return launch_kv_plan(*p, (hipStream_t)stream);
}

int flh_rope_table_create(uint32_t n_rot, uint32_t first, int layout, double base, const double * freq, uint32_t n_axis,
                          const uint8_t * axis, flh_rope_table ** out) {
    if (!out) return set_error(FLH_ERR_ARG, "rope table: null out");
    if (n_rot < 2 || n_rot > 1024 || n_rot % 2 || first > 65535)
        return set_error(FLH_ERR_ARG, "rope table: n_rot must be even, 2 .. 1024, first at most 65535");
    if (layout != FLH_ROPE_HALVES && layout != FLH_ROPE_PAIRS) return set_error(FLH_ERR_ARG, "rope table: unknown layout");
    if (n_axis < 1 || n_axis > 8) return set_error(FLH_ERR_ARG, "rope table: n_axis must be in 1 .. 8");
    if (!freq && !(base > 0 && isfinite(base))) return set_error(FLH_ERR_ARG, "rope table: base must be positive and finite");
    const uint32_t P = n_rot / 2;
    RopePair host[512];
    for (uint32_t i = 0; i < P; ++i) {
        const long double f = freq ? (long double)freq[i] : powl((long double)base, -(long double)(2 * i) / n_rot);
        if (!isfinite((double)f)) return set_error(FLH_ERR_ARG, "rope table: frequencies must be finite");
        if (axis && axis[i] >= n_axis) return set_error(FLH_ERR_ARG, "rope table: axis out of range");
        long double t = f / (2 * 3.14159265358979323846264338327950288L);
        t -= floorl(t);                                           // [0, 1]
        const long double w = roundl(ldexpl(t, 64));
        host[i] = RopePair{w >= 0x1p64L ? 0 : (uint64_t)w, axis ? axis[i] : 0u, 0u};
    }
    if (int rc = need_device()) return rc;
    flh_rope_table * r = new (std::nothrow) flh_rope_table{nullptr, n_rot, first, layout == FLH_ROPE_HALVES ? 1u : 0u};
    if (!r) return set_error(FLH_ERR_NOMEM, "rope table: out of memory");
    if (hipMalloc((void **)&r->dev, P * sizeof(RopePair)) != hipSuccess) {
        delete r;
        return set_error(FLH_ERR_NOMEM, "rope table: hipMalloc failed");
    }
    if (int rc = hip_check(hipMemcpy(r->dev, host, P * sizeof(RopePair), hipMemcpyHostToDevice), "rope table upload")) {
        (void)hipFree(r->dev);
        delete r;
        return rc;
    }
    *out = r;
    return FLH_OK;
}
int flh_rope_table_destroy(flh_rope_table * r) {
    if (!r) return FLH_OK;
    const int rc = hip_check(hipFree(r->dev), "rope table hipFree");
    delete r;
    return rc;
}

int flh_rope(const flh_rope_table * r, uint32_t dtype, const void * x, uint64_t x_tok, uint64_t x_head, void * y,
             uint64_t y_tok, uint64_t y_head, uint32_t n_tok, uint32_t n_head, uint32_t d, const int32_t * pos,
             uint32_t pos_stride, void * stream) {
    if (!r) return set_error(FLH_ERR_ARG, "rope: null table");
    if (dtype > FLH_DT_BF16) return set_error(FLH_ERR_ARG, "rope: unknown dtype");
    if (d == 0 || d > 65536 || n_head > 65535) return set_error(FLH_ERR_ARG, "rope: d must be in 1 .. 65536, n_head at most 65535");
    if (n_tok && n_head) {
        if (int rc = check_rope(r, d, pos)) return rc;
        if (int rc = check_turned(x, x_tok, x_head, y, y_tok, y_head, n_tok, n_head, d, dtype)) return rc;
    }
    if (int rc = need_device()) return rc;
    if (n_tok == 0 || n_head == 0) return FLH_OK;
    RopeArgs a{};
    set_rope(a, r);
    a.q = x; a.qo = y; a.q_tok = x_tok; a.q_head = x_head; a.qo_tok = y_tok; a.qo_head = y_head;
    a.n_tok = n_tok; a.n_head = n_head; a.d = d; a.pos = pos; a.pos_stride = pos_stride;
    const StreamTurn turn(stream);
    return launch_rope(a, dtype, FLH_DT_F16, (hipStream_t)stream);
}

int flh_rope_kv_append(const flh_rope_table * r, const flh_kv_cache * c, const flh_rope_kv_p * p, void * stream) {
    if (int rc = check_kv_cache(c)) return rc;
    if (!p) return set_error(FLH_ERR_ARG, "rope append: null arguments");
    if (p->dtype > FLH_DT_BF16) return set_error(FLH_ERR_ARG, "rope append: unknown dtype");
    if (p->n_head > 65535) return set_error(FLH_ERR_ARG, "rope append: n_head must be at most 65535");
    const uintptr_t el = elem(p->dtype);
    if (p->n_tok) {
        if (!p->k || !p->v || off(p->k, el) || off(p->v, el))
            return set_error(FLH_ERR_ARG, "rope append: k and v must be non-null and element aligned");
        if (!p->slot || off(p->slot, 4)) return set_error(FLH_ERR_ARG, "rope append: slot must be non-null and 4-byte aligned");
        if (int rc = check_rope(r, c->d_k, p->pos)) return rc;
        if (p->n_head)
            if (int rc = check_turned(p->q, p->q_tok, p->q_head, p->q_out, p->qo_tok, p->qo_head, p->n_tok, p->n_head, c->d_k,
                                      p->dtype)) return rc;
    }
    if (int rc = need_device()) return rc;
    if (p->n_tok == 0) return FLH_OK;
    RopeArgs a{};
    set_rope(a, r);
    a.q = p->q; a.qo = p->q_out; a.k = p->k; a.v = p->v; a.kc = c->k; a.vc = c->v; a.pos = p->pos; a.slot = p->slot;
    a.q_tok = p->q_tok; a.q_head = p->q_head; a.qo_tok = p->qo_tok; a.qo_head = p->qo_head;
    a.k_tok = p->k_tok; a.k_head = p->k_head; a.v_tok = p->v_tok; a.v_head = p->v_head;
    a.kc_page = c->k_page; a.kc_tok = c->k_tok; a.kc_head = c->k_head;
    a.vc_page = c->v_page; a.vc_tok = c->v_tok; a.vc_head = c->v_head;
    a.n_tok = p->n_tok; a.n_head = p->n_head; a.n_kv = c->n_kv_head; a.d = c->d_k; a.dv = c->d_v;
    a.pos_stride = p->pos_stride; a.n_slot = c->n_pages * c->page_size; a.sh = (uint32_t)__builtin_ctz(c->page_size);
    const StreamTurn turn(stream);
    return launch_rope(a, p->dtype, c->dtype, (hipStream_t)stream);
}

size_t flh_paged_attn_ws_bytes(const flh_kv_cache * c, const flh_attn_p * p) {
    AttnTreeArgs a;
    if (attn_args(c, p, a)) return 0;
    return attn_ws_bytes(a, p->dtype);
}

int flh_paged_attn(const flh_kv_cache * c, const flh_attn_p * p, void * stream) {
    AttnTreeArgs a;
    if (int rc = attn_args(c, p, a)) return rc;
    return attn_run(c, p, a, stream);
}

size_t flh_tree_attn_ws_bytes(const flh_kv_cache * c, const flh_attn_p * p) {
    AttnTreeArgs a;
    if (attn_args(c, p, a)) return 0;
    a.tree_stride = 1;
    return attn_ws_bytes(a, p->dtype);
}

int flh_tree_attn(const flh_kv_cache * c, const flh_attn_p * p, const flh_tree_p * t, void * stream) {
    AttnTreeArgs a;
    if (int rc = attn_args(c, p, a)) return rc;
    if (!t) return set_error(FLH_ERR_ARG, "tree attention: null arguments");
    if (!p->causal) return set_error(FLH_ERR_ARG, "tree attention: causal must be set");
    if (t->mask_stride == 0 || t->mask_stride > 32768) return set_error(FLH_ERR_ARG, "tree attention: mask_stride must be in 1 .. 32768");
    if (p->n_tok && p->n_seq) {
        if (!t->mask || off(t->mask, 4)) return set_error(FLH_ERR_ARG, "tree attention: mask must be non-null and 4-byte aligned");
        if ((p->window && !t->depth) || off(t->depth, 4))
            return set_error(FLH_ERR_ARG, "tree attention: a window needs depth, 4-byte aligned");
    }
    a.tree_mask = t->mask; a.tree_depth = t->depth; a.tree_stride = t->mask_stride;
    return attn_run(c, p, a, stream);
}

}  // extern "C"
