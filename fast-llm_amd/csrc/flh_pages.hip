// flh_pages.hip -- the paged cache's pages between steps: requests forked (full pages are
// shared, a partly filled one is copied), cut back and freed, and tokens moved into place in all layers.
#include "flh_common.h"
#include "flh_internal.h"
#include "flh_status.h"

namespace flh {

constexpr uint32_t PG_T = 1024;

// exclusive scan of v over the workgroup (ws: 16 wave sums); total in *sum
__device__ __forceinline__ uint32_t scan_before(uint32_t v, uint32_t * ws, uint32_t * sum) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t in = v;
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_up(in, d);
        if (lane >= d) in += o;
    }
    __syncthreads();                                              // ws may hold the scan before
    if (lane == 63) ws[wave] = in;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (uint32_t w = 0; w < PG_T / 64; ++w) {
        if (w < wave) before += ws[w];
        all += ws[w];
    }
    *sum = all;
    return before + in - v;
}

// ------------------------------------------------------------------- fork --
// Workgroup 0 gives the forks their lengths and the partly filled pages their
// copies (a scan over the forks, 1024 at a time); the others copy a fork's full pages each and count
// one holder more for them.  A launch and a round of loads: 8 forks of 126 pages 3.4 us, 128 of up to 24 4.8.
__global__ __launch_bounds__(PG_T) void k_kv_fork(flh_kv_fork_p p, uint32_t sh) {
    __shared__ uint32_t ws[PG_T / 64];
    const uint32_t tid = threadIdx.x, ps = 1u << sh;
    // tokens that fork f takes over (false: no such request)
    auto job = [&](uint32_t f, uint32_t & src, uint32_t & dst, uint32_t & len) {
        src = p.src[f];
        dst = p.dst[f];
        if (src >= p.n_seq || dst >= p.n_seq || src == dst) return false;
        len = min(p.kv_len[src], p.len ? p.len[f] : 0xFFFFFFFFu);
        len = (uint32_t)min((uint64_t)len, (uint64_t)p.table_stride << sh);
        return true;
    };
    if (blockIdx.x) {
        uint32_t src, dst, len;
        if (!job(blockIdx.x - 1, src, dst, len)) return;
        const uint32_t * from = p.table + (uint64_t)src * p.table_stride;
        uint32_t * to = p.table + (uint64_t)dst * p.table_stride;
        for (uint32_t j = blockIdx.y * PG_T + tid; j < len >> sh; j += gridDim.y * PG_T) {
            const uint32_t e = from[j];
            to[j] = e < p.n_pages ? e : FLH_KV_NONE;
            if (e < p.n_pages) atomicAdd(p.shared + e, 1u);
        }
        return;
    }
    if (blockIdx.y) return;
    uint32_t taken = *p.taken, copies = 0, none = 0;
    for (uint32_t f0 = 0; f0 < p.n_fork; f0 += PG_T) {
        const uint32_t f = f0 + tid;
        uint32_t src = 0, dst = 0, len = 0, last = FLH_KV_NONE, fresh = FLH_KV_NONE;
        const bool on = f < p.n_fork && job(f, src, dst, len);
        const uint32_t full = len >> sh, part = on ? len & (ps - 1) : 0;
        if (part) last = p.table[(uint64_t)src * p.table_stride + full];
        const uint32_t need = part && last < p.n_pages;
        uint32_t sum;
        const uint64_t at = (uint64_t)taken + scan_before(need, ws, &sum);
        if (need && at < p.n_free) fresh = p.free_pages[at];
        const bool got = fresh < p.n_pages;
        if (on) {
            if (part) p.table[(uint64_t)dst * p.table_stride + full] = got ? fresh : FLH_KV_NONE;
            p.kv_len[dst] = len;
        }
        if (f < p.n_fork) {
            p.copy_src[f] = got ? last << sh : FLH_KV_NONE;
            p.copy_dst[f] = got ? fresh << sh : FLH_KV_NONE;
            p.copy_n[f] = got ? part : 0;
        }
        taken = taken > 0xFFFFFFFFu - sum ? 0xFFFFFFFFu : taken + sum;
        copies += __syncthreads_count(got);
        none += __syncthreads_count(need && !got);
    }
    if (tid == 0) {
        *p.taken = taken;
        if (p.info) {
            p.info[0] = copies;
            p.info[1] = none;
        }
    }
}

int launch_kv_fork(const flh_kv_fork_p & p, hipStream_t s) {
    const uint32_t sh = (uint32_t)__builtin_ctz(p.page_size);
    // (a workgroup copies 1024 entries a turn; more of them for a fork where forks are few)
    const uint32_t parts = std::max(1u, std::min((p.table_stride + PG_T - 1) / PG_T, 256 / p.n_fork));
    hipLaunchKernelGGL(k_kv_fork, dim3(p.n_fork + 1, parts), dim3(PG_T), 0, s, p, sh);
    return hip_check(hipGetLastError(), "k_kv_fork launch");
}

// ------------------------------------------------------------------- trim --
// One workgroup walks the requests 1024 at a time, and the pages that they leave flat, four a
// thread and turn.  A page is put back by the last holder that leaves it, in the order of requests and pages,
// not of time: all count themselves off first (below 0: nobody holds it any more), then the
// place of the last one in order is found by a minimum in the page's own count, which that one makes 0 again
// when it puts the page back.  Without counts every page left is put back.  Rounds of loads and of
// atomics bound it; up to 4096 pages of up to 1024 requests, what a step leaves, are found once and stay in registers (8 forks
// of 126 pages each 10.2 us, 18.0 found again in each round; 64 requests of 3 pages 7.0, 13.4).  Many more take a
// microsecond for about 90 pages (8192 pages 94 us), 700 without counts.
struct TrimOf {
    uint32_t before, after, part;       // pages held, pages kept, tokens in a last one that is partly filled
};
__device__ __forceinline__ TrimOf trim_of(const flh_kv_trim_p & p, uint32_t held, uint32_t keep, uint32_t sh) {
    const uint64_t ps = 1ull << sh, all = ((uint64_t)keep + ps - 1) >> sh;
    TrimOf t;
    t.before = (uint32_t)min(((uint64_t)held + ps - 1) >> sh, (uint64_t)p.table_stride);
    t.after = (uint32_t)min(all, (uint64_t)p.table_stride);
    t.part = all <= p.table_stride ? keep & (uint32_t)(ps - 1) : 0;
    return t;
}

__global__ __launch_bounds__(PG_T) void k_kv_trim(flh_kv_trim_p p, uint32_t sh) {
    constexpr uint32_t N = 4;
    __shared__ uint32_t ws[PG_T / 64], l_at[PG_T], l_from[PG_T], l_own[PG_T];
    const uint32_t tid = threadIdx.x;
    const bool once = p.n_seq <= PG_T;
    uint32_t taken = min(*p.taken, p.n_free), lost = 0, sum = 0;
    // A batch of requests: where their pages are on the line of all that are left (l_at), from which table entry on; l_own: a
    // last page that others hold too, which is left, too, and has a fresh one in its place (before anybody leaves a page)
    auto batch = [&](uint32_t s0, bool first) {
        const uint32_t s = s0 + tid;
        uint32_t own = FLH_KV_NONE;
        TrimOf t{0, 0, 0};
        if (s < p.n_seq) {
            const uint32_t held = p.kv_len[s];
            t = trim_of(p, held, min(held, p.keep[s]), sh);
        }
        if (p.shared && first) {
            uint32_t * at = p.table + (uint64_t)s * p.table_stride + (t.after - 1);
            uint32_t last = FLH_KV_NONE, fresh = FLH_KV_NONE;
            if (t.part) last = *at;
            const bool need = last < p.n_pages && p.shared[last] != 0;
            const uint32_t i = taken + scan_before(need, ws, &sum);
            if (need && i < p.n_free) fresh = p.free_pages[i];
            const bool got = fresh < p.n_pages;
            if (s < p.n_seq) {
                p.copy_src[s] = need ? last << sh : FLH_KV_NONE;  // (without a page to go to: until the end)
                p.copy_dst[s] = got ? fresh << sh : FLH_KV_NONE;
                p.copy_n[s] = got ? t.part : 0;
                if (need) *at = got ? fresh : FLH_KV_NONE;
            }
            if (need) own = last;
            lost += __syncthreads_count(need && !got);
            taken = min(p.n_free, taken + sum);
        } else if (p.shared && s < p.n_seq) {
            own = p.copy_src[s];
            if (own != FLH_KV_NONE) own >>= sh;
        }
        const uint32_t at = scan_before(t.before - t.after + (own != FLH_KV_NONE), ws, &sum);
        l_at[tid] = at;
        l_from[tid] = t.after;
        l_own[tid] = own;
        __syncthreads();
    };
    // entry i of the batch's line: the page, and its place in the table (null: none)
    auto entry = [&](uint32_t s0, uint32_t i, uint32_t & e, uint32_t *& in) {
        e = FLH_KV_NONE;
        in = nullptr;
        if (i >= sum) return;
        uint32_t lo = 0, n = min(PG_T, p.n_seq - s0);
        while (n > 1) {
            const uint32_t h = n >> 1;
            if (l_at[lo + h] <= i) { lo += h; n -= h; }
            else n = h;
        }
        const uint32_t j = i - l_at[lo], own = l_own[lo];
        if (own != FLH_KV_NONE && j == 0) e = own;
        else {
            in = p.table + (uint64_t)(s0 + lo) * p.table_stride + l_from[lo] + j - (own != FLH_KV_NONE);
            e = *in;
        }
    };
    uint32_t e[N];
    uint32_t * in[N];
    bool kept = false;
    // with(i, page, place) for every page that is left, i its place in the order of all; all threads together
    auto each = [&](auto && with) {
        if (kept) {
#pragma unroll
            for (uint32_t k = 0; k < N; ++k)
                if (k * PG_T < sum) with(k * PG_T + tid, e[k], in[k]);
        } else {
            uint32_t base = 0;
            for (uint32_t s0 = 0; s0 < p.n_seq; s0 += PG_T) {
                if (!once) batch(s0, false);
                for (uint32_t i0 = 0; i0 < sum; i0 += N * PG_T) {
#pragma unroll
                    for (uint32_t k = 0; k < N; ++k) entry(s0, i0 + k * PG_T + tid, e[k], in[k]);
#pragma unroll
                    for (uint32_t k = 0; k < N; ++k)
                        if (i0 + k * PG_T < sum) with(base + i0 + k * PG_T + tid, e[k], in[k]);
                }
                base += sum;
                __syncthreads();                                  // the tables in LDS are the next batch's
            }
        }
        __threadfence_block();
        __syncthreads();
    };
    for (uint32_t s0 = 0; s0 < p.n_seq; s0 += PG_T)
        if (once || p.shared) {
            batch(s0, true);
            __syncthreads();
        }
    if (once && sum <= N * PG_T) {
#pragma unroll
        for (uint32_t k = 0; k < N; ++k) entry(0, k * PG_T + tid, e[k], in[k]);
        kept = true;
    }
    int32_t * count = (int32_t *)p.shared;
    if (p.shared) {
        each([&](uint32_t, uint32_t x, uint32_t *) { if (x < p.n_pages) atomicSub(count + x, 1); });
        // (-2 - the last one's place is below the count, also of a page that was left more often than it was held: places
        // are as many)
        each([&](uint32_t i, uint32_t x, uint32_t *) {
            if (x < p.n_pages && __hip_atomic_load(count + x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) < 0)
                atomicMin(count + x, -2 - (int32_t)i);
        });
    }
    // ---- put back, one after another: the last one is taken next
    uint32_t back = 0;
    each([&](uint32_t i, uint32_t x, uint32_t * at) {
        bool mine = x < p.n_pages;
        if (p.shared && mine) {
            mine = __hip_atomic_load(count + x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == -2 - (int32_t)i;
            if (mine) __hip_atomic_store(count + x, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        uint32_t all;
        const uint32_t to = back + scan_before(mine, ws, &all);
        if (mine && to < taken) p.free_pages[taken - 1 - to] = x;
        if (at) *at = FLH_KV_NONE;
        back += all;
    });
    for (uint32_t s = tid; s < p.n_seq; s += PG_T) {
        p.held[s] = min(p.kv_len[s], p.keep[s]);
        if (p.shared && p.copy_dst[s] == FLH_KV_NONE) p.copy_src[s] = FLH_KV_NONE;
    }
    if (tid == 0) {
        *p.taken = taken - min(back, taken);
        if (p.info) {
            p.info[0] = min(back, taken);
            p.info[1] = lost + back - min(back, taken);
        }
    }
}

int launch_kv_trim(const flh_kv_trim_p & p, hipStream_t s) {
    hipLaunchKernelGGL(k_kv_trim, dim3(1), dim3(PG_T), 0, s, p, (uint32_t)__builtin_ctz(p.page_size));
    return hip_check(hipGetLastError(), "k_kv_trim launch");
}

// -------------------------------------------------------------------- move --
// A thread owns 16 bytes of a token's keys or values in one layer (its place is found once) and
// carries them from slot to slot, several tokens at once (8 loads on their way a thread).  Bytes bound it where there are
// many: 128 copies of up to 64 tokens in 16 layers 80 us (491 MB read and written, 6.1 TB/s: a source that several forks
// copy comes from the last-level cache); 8 of 9 tokens in 32 layers 5.7, 64 paths in trees of up to 25 rows 11.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
constexpr uint32_t MV_T = 256, MV_LAYERS = 64, MV_GRID = 65535;   // (the grid's second axis)
struct MoveArgs {
    uint8_t * k[MV_LAYERS]; uint8_t * v[MV_LAYERS];
    uint64_t k_page, k_tok, k_head, v_page, v_tok, v_head;      // strides in bytes
    uint32_t n_cache, n_head, pk, pv, n_slot, sh;               // pieces of 16 bytes of a head's keys and values
    uint32_t units;                                             // pieces of a token: n_head * (pk + pv)
};
struct MoveLane {
    uint8_t * at;
    uint64_t page, tok;
    uint32_t sh;
    __device__ __forceinline__ u32x4 * of(uint32_t slot) const {
        return (u32x4 *)(at + (uint64_t)(slot >> sh) * page + (uint64_t)(slot & ((1u << sh) - 1u)) * tok);
    }
};
// piece g of the layers' tokens (g < n_cache * units)
__device__ __forceinline__ MoveLane move_lane(const MoveArgs & a, uint32_t g) {
    const uint32_t c = g / a.units, u = g - c * a.units, nk = a.n_head * a.pk;
    const bool isk = u < nk;
    const uint32_t x = isk ? u : u - nk, per = isk ? a.pk : a.pv, h = x / per;
    return MoveLane{(isk ? a.k[c] : a.v[c]) + h * (isk ? a.k_head : a.v_head) + (uint64_t)(x - h * per) * 16,
                    isk ? a.k_page : a.v_page, isk ? a.k_tok : a.v_tok, a.sh};
}

// Copy y: n tokens from a slot on to another one on, inside a page each.
__global__ __launch_bounds__(MV_T) void k_kv_copy(MoveArgs a, const uint32_t * src, const uint32_t * dst, const uint32_t * count) {
    const uint32_t i = blockIdx.y, from = src[i], to = dst[i], ps = 1u << a.sh;
    if (from >= a.n_slot || to >= a.n_slot) return;
    const uint32_t n = min(count[i], min(ps - (from & (ps - 1)), ps - (to & (ps - 1))));
    const uint32_t g = blockIdx.x * MV_T + threadIdx.x;
    if (g >= a.n_cache * a.units) return;
    const MoveLane l = move_lane(a, g);
    constexpr uint32_t N = 8;
    for (uint32_t t = blockIdx.z * N; t < n; t += gridDim.z * N) {
        u32x4 x[N];                                              // (behind the last one: that one again)
#pragma unroll
        for (uint32_t j = 0; j < N; ++j) x[j] = *l.of(from + min(t + j, n - 1));
#pragma unroll
        for (uint32_t j = 0; j < N; ++j)
            if (t + j < n) *l.of(to + t + j) = x[j];
    }
}

// Request y: token path[j] into token j's place, in ascending order.  A place is only
// written when the token that stood there has been read: path[j] >= j ascends, so the place of j
// is that of no later path[k], and a thread reads a token before it writes it and those behind it.
__global__ __launch_bounds__(MV_T) void k_kv_compact(MoveArgs a, flh_kv_compact_p p) {
    constexpr uint32_t N = 8;
    __shared__ uint32_t from[MV_T], to[MV_T];
    const uint32_t s = blockIdx.y, r0 = min(p.q_start[s], p.n_tok), r1 = min(p.q_start[s + 1], p.n_tok);
    const uint32_t rows = r1 > r0 ? r1 - r0 : 0, n = min(min(p.n_path[s], p.path_stride), rows);
    const uint32_t g = blockIdx.x * MV_T + threadIdx.x;
    const bool on = g < a.n_cache * a.units;
    const MoveLane l = move_lane(a, on ? g : 0);
    for (uint32_t j0 = 0; j0 < n; j0 += MV_T) {
        const uint32_t j = j0 + threadIdx.x, m = min(n - j0, MV_T);
        uint32_t x = FLH_KV_NONE, y = FLH_KV_NONE;
        if (j < n) {
            const uint32_t r = p.path[(uint64_t)s * p.path_stride + j];
            if (r > j && r < rows) {                             // (r == j: it stands where it is)
                x = p.slot[r0 + r];
                y = p.slot[r0 + j];
            }
        }
        const bool move = x < a.n_slot && y < a.n_slot && x != y;
        __syncthreads();
        from[threadIdx.x] = move ? x : FLH_KV_NONE;
        to[threadIdx.x] = y;
        __syncthreads();
        if (!on) continue;
        for (uint32_t t = 0; t < m; t += N) {
            u32x4 v[N];
            uint32_t x[N], y[N];
#pragma unroll
            for (uint32_t i = 0; i < N; ++i) {
                const uint32_t at = min(t + i, m - 1);
                x[i] = from[at];
                y[i] = t + i < m && x[i] != FLH_KV_NONE ? to[at] : FLH_KV_NONE;
                v[i] = *l.of(x[i] != FLH_KV_NONE ? x[i] : 0u);    // (slot 0: any that is there)
            }
#pragma unroll
            for (uint32_t i = 0; i < N; ++i)
                if (y[i] != FLH_KV_NONE) *l.of(y[i]) = v[i];
        }
    }
}

// Calls `with` for every MV_LAYERS layers
template <typename F> static int by_layers(const flh_kv_cache * c, uint32_t n, F && with) {
    MoveArgs a{};
    a.k_page = 2 * c->k_page; a.k_tok = 2 * c->k_tok; a.k_head = 2 * c->k_head;
    a.v_page = 2 * c->v_page; a.v_tok = 2 * c->v_tok; a.v_head = 2 * c->v_head;
    a.n_head = c->n_kv_head; a.pk = c->d_k / 8; a.pv = c->d_v / 8; a.units = a.n_head * (a.pk + a.pv);
    a.n_slot = c->n_pages * c->page_size; a.sh = (uint32_t)__builtin_ctz(c->page_size);
    for (uint32_t i = 0; i < n; i += MV_LAYERS) {
        a.n_cache = std::min(n - i, MV_LAYERS);
        for (uint32_t j = 0; j < a.n_cache; ++j) {
            a.k[j] = (uint8_t *)c[i + j].k;
            a.v[j] = (uint8_t *)c[i + j].v;
        }
        if (int rc = with(a, (a.n_cache * a.units + MV_T - 1) / MV_T)) return rc;
    }
    return FLH_OK;
}
int launch_kv_copy(const flh_kv_cache * c, uint32_t n, const uint32_t * src, const uint32_t * dst, const uint32_t * count,
                   uint32_t n_copy, hipStream_t s) {
    return by_layers(c, n, [&](const MoveArgs & a, uint32_t wgs) -> int {
        // (where there are few copies, a page's tokens are shared by several workgroups)
        const uint32_t parts = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>((c->page_size + 7) / 8, 2048 / ((uint64_t)wgs * n_copy)));
        for (uint32_t i = 0; i < n_copy; i += MV_GRID) {
            const uint32_t m = std::min(n_copy - i, MV_GRID);
            hipLaunchKernelGGL(k_kv_copy, dim3(wgs, m, parts), dim3(MV_T), 0, s, a, src + i, dst + i, count + i);
            if (int rc = hip_check(hipGetLastError(), "k_kv_copy launch")) return rc;
        }
        return FLH_OK;
    });
}
int launch_kv_compact(const flh_kv_cache * c, uint32_t n, const flh_kv_compact_p & p, hipStream_t s) {
    return by_layers(c, n, [&](const MoveArgs & a, uint32_t wgs) -> int {
        for (uint32_t i = 0; i < p.n_seq; i += MV_GRID) {
            flh_kv_compact_p q = p;
            q.q_start += i;
            q.n_path += i;
            q.path += (uint64_t)i * p.path_stride;
            hipLaunchKernelGGL(k_kv_compact, dim3(wgs, std::min(p.n_seq - i, MV_GRID)), dim3(MV_T), 0, s, a, q);
            if (int rc = hip_check(hipGetLastError(), "k_kv_compact launch")) return rc;
        }
        return FLH_OK;
    });
}

}  // namespace flh
