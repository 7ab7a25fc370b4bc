// flh_spec.cpp -- entry points of drafted trees, their verification and the pages between
// steps (include/fastllm_hip.h): argument checks, then one call of the launchers.  Nothing is
// launched on an error.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <initializer_list>
#include "../../include/fastllm_hip.h"
#include "flh_internal.h"
#include "flh_status.h"

using namespace flh;

namespace {

bool off(const void * p, uintptr_t align) { return ((uintptr_t)p & (align - 1)) != 0; }
bool any_null(std::initializer_list<const void *> ps) {
    for (const void * p : ps)
        if (!p) return true;
    return false;
}
bool any_off(std::initializer_list<const void *> ps) {
    for (const void * p : ps)
        if (off(p, 4)) return true;
    return false;
}
bool pow2_page(uint32_t n) { return n >= 1 && n <= 65536 && (n & (n - 1)) == 0; }

int check_verify(const flh_verify_p * p) {
    if (!p) return set_error(FLH_ERR_ARG, "verify: null arguments");
    if (p->dtype > FLH_DT_BF16) return set_error(FLH_ERR_ARG, "verify: unknown dtype");
    if (p->vocab == 0 || p->vocab > (1u << 22)) return set_error(FLH_ERR_UNSUPPORTED, "verify: vocab must be in 1 .. 2^22");
    if (p->path_stride == 0) return set_error(FLH_ERR_ARG, "verify: path_stride must be at least 1");
    if (p->max_child == 0 || p->max_child > 64) return set_error(FLH_ERR_ARG, "verify: max_child must be in 1 .. 64");
    const uint64_t chunks = (p->vocab + 4095) / 4096;             // (a grid's threads are counted in 32 bits)
    if (p->n_tok * chunks >= (1u << 24) || p->n_seq * chunks >= (1u << 24))
        return set_error(FLH_ERR_UNSUPPORTED, "verify: too many rows for one call");
    return FLH_OK;
}

int check_caches(const flh_kv_cache * c, uint32_t n) {
    if (n && !c) return set_error(FLH_ERR_ARG, "kv caches: null");
    for (uint32_t i = 0; i < n; ++i) {
        if (int rc = check_kv_cache(c + i)) return rc;
        const flh_kv_cache & a = c[0], & b = c[i];
        if (a.dtype != b.dtype || a.n_pages != b.n_pages || a.page_size != b.page_size || a.n_kv_head != b.n_kv_head ||
            a.d_k != b.d_k || a.d_v != b.d_v || a.k_page != b.k_page || a.k_tok != b.k_tok || a.k_head != b.k_head ||
            a.v_page != b.v_page || a.v_tok != b.v_tok || a.v_head != b.v_head)
            return set_error(FLH_ERR_ARG, "kv caches: they must be alike but for k and v");
    }
    return FLH_OK;
}

int check_pages(uint32_t n_pages, uint32_t page_size) {
    if (!pow2_page(page_size)) return set_error(FLH_ERR_UNSUPPORTED, "kv pages: page_size must be a power of two up to 65536");
    if ((uint64_t)n_pages * page_size >= 0xFFFFFFFFull) return set_error(FLH_ERR_ARG, "kv pages: n_pages * page_size must be below 2^32 - 1");
    return FLH_OK;
}

}  // namespace

extern "C" {

int flh_tree_plan(const flh_tree_plan_p * p, void * stream) {
    if (!p) return set_error(FLH_ERR_ARG, "tree plan: null arguments");
    if (p->mask_stride == 0 || p->mask_stride > 32768) return set_error(FLH_ERR_ARG, "tree plan: mask_stride must be in 1 .. 32768");
    // (a chain of all rows is walked up by each of them for each word: at this size for some seconds)
    if (p->n_tok > (1u << 22) || (uint64_t)p->n_tok * p->n_tok * p->mask_stride > (1ull << 44))
        return set_error(FLH_ERR_UNSUPPORTED, "tree plan: n_tok * n_tok * mask_stride must be at most 2^44");
    if (p->n_tok && p->n_seq && (any_null({p->q_start, p->parent, p->mask, p->depth}) || (p->pos && !p->kv_len)))
        return set_error(FLH_ERR_ARG, "tree plan: null argument");
    if (any_off({p->q_start, p->parent, p->kv_len, p->mask, p->depth, p->pos}))
        return set_error(FLH_ERR_ARG, "tree plan: arrays must be 4-byte aligned");
    if (int rc = need_device()) return rc;
    if (p->n_tok == 0 || p->n_seq == 0) return FLH_OK;
    const StreamTurn turn(stream);
    return launch_tree_plan(*p, (hipStream_t)stream);
}

size_t flh_spec_verify_ws_bytes(const flh_verify_p * p) { return check_verify(p) ? 0 : verify_ws_bytes(*p); }

int flh_spec_verify(const flh_verify_p * p, void * stream) {
    if (int rc = check_verify(p)) return rc;
    if (p->n_seq) {
        if (any_null({p->q_start, p->u_next, p->n_path, p->path, p->next}) || (p->n_tok && any_null({p->target, p->token, p->u_accept})) ||
            (p->len && !p->kv_len))
            return set_error(FLH_ERR_ARG, "verify: null argument");
        if (any_off({p->q_start, p->token, p->parent, p->inv_temp, p->u_accept, p->u_next, p->kv_len, p->n_path, p->path, p->next,
                     p->logp, p->len}))
            return set_error(FLH_ERR_ARG, "verify: arrays must be 4-byte aligned");
        const uintptr_t el = p->dtype == FLH_DT_F32 ? 4 : 2;
        if (off(p->target, el) || off(p->draft, el)) return set_error(FLH_ERR_ARG, "verify: logits must be element aligned");
        const size_t need = verify_ws_bytes(*p);
        if (need && (!p->ws || off(p->ws, 16) || p->ws_bytes < need))
            return set_error(FLH_ERR_ARG, "verify: ws must be 16-byte aligned and of flh_spec_verify_ws_bytes");
    }
    if (int rc = need_device()) return rc;
    if (p->n_seq == 0) return FLH_OK;
    const StreamTurn turn(stream, true);                          // (launches that pass the workspace on)
    return launch_verify(*p, (hipStream_t)stream);
}

int flh_kv_compact(const flh_kv_cache * caches, uint32_t n_cache, const flh_kv_compact_p * p, void * stream) {
    if (int rc = check_caches(caches, n_cache)) return rc;
    if (!p) return set_error(FLH_ERR_ARG, "kv compact: null arguments");
    if (p->n_seq && p->n_tok && p->path_stride && any_null({p->q_start, p->slot, p->n_path, p->path}))
        return set_error(FLH_ERR_ARG, "kv compact: null argument");
    if (any_off({p->q_start, p->slot, p->n_path, p->path})) return set_error(FLH_ERR_ARG, "kv compact: arrays must be 4-byte aligned");
    if (int rc = need_device()) return rc;
    if (p->n_seq == 0 || p->n_tok == 0 || p->path_stride == 0 || n_cache == 0) return FLH_OK;
    const StreamTurn turn(stream, n_cache > 64 || p->n_seq > 65535);
    return launch_kv_compact(caches, n_cache, *p, (hipStream_t)stream);
}

int flh_kv_copy(const flh_kv_cache * caches, uint32_t n_cache, const uint32_t * src, const uint32_t * dst, const uint32_t * n_tok,
                uint32_t n_copy, void * stream) {
    if (int rc = check_caches(caches, n_cache)) return rc;
    if (n_copy && any_null({src, dst, n_tok})) return set_error(FLH_ERR_ARG, "kv copy: null argument");
    if (any_off({src, dst, n_tok})) return set_error(FLH_ERR_ARG, "kv copy: arrays must be 4-byte aligned");
    if (int rc = need_device()) return rc;
    if (n_copy == 0 || n_cache == 0) return FLH_OK;
    const StreamTurn turn(stream, n_cache > 64 || n_copy > 65535);
    return launch_kv_copy(caches, n_cache, src, dst, n_tok, n_copy, (hipStream_t)stream);
}

int flh_kv_fork(const flh_kv_fork_p * p, void * stream) {
    if (!p) return set_error(FLH_ERR_ARG, "kv fork: null arguments");
    if (int rc = check_pages(p->n_pages, p->page_size)) return rc;
    if (p->n_fork > (1u << 21)) return set_error(FLH_ERR_UNSUPPORTED, "kv fork: n_fork must be at most 2^21");
    if (p->n_fork && (any_null({p->src, p->dst, p->kv_len, p->table, p->taken, p->shared, p->copy_src, p->copy_dst, p->copy_n}) ||
                      (p->n_free && !p->free_pages) || p->table_stride == 0))
        return set_error(FLH_ERR_ARG, "kv fork: null argument");
    if (any_off({p->src, p->dst, p->len, p->kv_len, p->table, p->free_pages, p->taken, p->shared, p->copy_src, p->copy_dst, p->copy_n, p->info}))
        return set_error(FLH_ERR_ARG, "kv fork: arrays must be 4-byte aligned");
    if (int rc = need_device()) return rc;
    if (p->n_fork == 0) return FLH_OK;
    const StreamTurn turn(stream);
    return launch_kv_fork(*p, (hipStream_t)stream);
}

int flh_kv_trim(const flh_kv_trim_p * p, void * stream) {
    if (!p) return set_error(FLH_ERR_ARG, "kv trim: null arguments");
    if (int rc = check_pages(p->n_pages, p->page_size)) return rc;
    if ((uint64_t)p->n_seq * p->table_stride >= (1ull << 31) - 1)
        return set_error(FLH_ERR_UNSUPPORTED, "kv trim: n_seq * table_stride must be below 2^31 - 1");
    if (p->n_seq && (any_null({p->kv_len, p->keep, p->held, p->table, p->taken}) || (p->n_free && !p->free_pages) || p->table_stride == 0 ||
                     (p->shared && any_null({p->copy_src, p->copy_dst, p->copy_n}))))
        return set_error(FLH_ERR_ARG, "kv trim: null argument");
    if (any_off({p->kv_len, p->keep, p->held, p->table, p->free_pages, p->taken, p->shared, p->copy_src, p->copy_dst, p->copy_n, p->info}))
        return set_error(FLH_ERR_ARG, "kv trim: arrays must be 4-byte aligned");
    if (int rc = need_device()) return rc;
    if (p->n_seq == 0) return FLH_OK;
    const StreamTurn turn(stream);
    return launch_kv_trim(*p, (hipStream_t)stream);
}

}  // extern "C"
