// flh_kv.hip -- the paged key/value cache's book-keeping and writes: block
// tables and slot maps from request lengths, rotary positions, and the append
// of keys and values.
#include "flh_common.h"
#include "flh_internal.h"
#include "flh_status.h"

namespace flh {

// ------------------------------------------------------------------- plan --
// One workgroup walks the requests 1024 at a time (thread per request): an
// exclusive scan of the new rows and of the pages needed, carried from batch to
// batch, gives every request its first row and its first entry of the free list;
// then the batch's new pages and (rows <= PLAN_ROWS) rows are dealt to the
// threads flat, each finding its request by a binary search over the scan in
// LDS.  More rows go to k_kv_slots, a launch over all CUs behind this one.  One
// workgroup, so taken and kv_len may be updated in place: nobody else reads
// them.  Sums are 64-bit (a garbage length costs its own rows only).  A launch and
// a chain of loads, scans and searches bound it: 64 requests of a token each take
// 7.0 us, 500 with 64000 rows 11.7 (two launches).  (A thread of 1024
// has 128 registers: five are spilled.)  Rows in the same launch cost one
// workgroup 1 us for about 1200 of them, a second launch 4 to 5 us: 2048 rows take 8.8
// us in one and 12.1 in two, 8192 13.4 and 12.2, 16384 19.9 and 12.1.
constexpr uint32_t PLAN_T = 1024;

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, uint32_t d) {
    const uint32_t lo = __shfl_up((uint32_t)v, d), hi = __shfl_up((uint32_t)(v >> 32), d);
    return ((uint64_t)hi << 32) | lo;
}
// inclusive scan of v over the workgroup (ws: 16 wave sums); total in *sum
__device__ __forceinline__ uint64_t scan_wg(uint64_t v, uint64_t * ws, uint64_t * sum) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) {
        const uint64_t o = shfl_up64(v, d);
        if (lane >= d) v += o;
    }
    __syncthreads();                                              // ws may hold the scan before
    if (lane == 63) ws[wave] = v;
    __syncthreads();
    uint64_t before = 0, all = 0;
#pragma unroll
    for (uint32_t w = 0; w < PLAN_T / 64; ++w) {
        if (w < wave) before += ws[w];
        all += ws[w];
    }
    *sum = all;
    return v + before;
}
__device__ __forceinline__ uint32_t sat32(uint64_t v) { return v > 0xFFFFFFFFull ? 0xFFFFFFFFu : (uint32_t)v; }

// the last of n requests (n >= 1) whose entry of the ascending at is <= i
template <typename T>
__device__ __forceinline__ uint32_t owner(const T * at, uint32_t n, T i) {
    uint32_t lo = 0;
    while (n > 1) {
        const uint32_t h = n >> 1;
        if (at[lo + h] <= i) { lo += h; n -= h; }
        else n = h;
    }
    return lo;
}
__device__ __forceinline__ uint32_t slot_of(uint32_t page, uint32_t at, uint32_t sh) {
    return page > (0xFFFFFFFEu >> sh) ? FLH_KV_NONE : (page << sh) | (at & ((1u << sh) - 1u));
}

// tokens [from, to) of a request, all in the page `page`, that have no slot
__device__ __forceinline__ uint32_t lost_in(uint32_t page, uint64_t from, uint64_t to, uint32_t sh) {
    if (slot_of(page, 0, sh) == FLH_KV_NONE) return (uint32_t)(to - from);
    return slot_of(page, (uint32_t)(to - 1), sh) == FLH_KV_NONE;  // (a page's last slot may be that number itself)
}

__global__ __launch_bounds__(PLAN_T) void k_kv_plan(flh_kv_plan_p p, uint32_t sh, int rows_too) {
    __shared__ uint64_t ws[PLAN_T / 64], l_page[PLAN_T];
    __shared__ uint32_t l_row[PLAN_T], l_rows[PLAN_T], l_held[PLAN_T], l_before[PLAN_T];
    const uint32_t tid = threadIdx.x;
    const uint64_t ps = 1ull << sh;
    uint64_t row0 = 0, page0 = p.taken_in ? *p.taken_in : 0, lost = 0;
    for (uint32_t base = 0; base < p.n_seq; base += PLAN_T) {
        const uint32_t s = base + tid, nb = min(PLAN_T, p.n_seq - base);
        const bool in = tid < nb;
        const uint64_t held = in ? p.held[s] : 0, add = in ? p.add[s] : 0;
        uint64_t sum;
        const uint64_t end = row0 + scan_wg(add, ws, &sum);
        const uint32_t r0 = (uint32_t)min(end - add, (uint64_t)p.max_tok), r1 = (uint32_t)min(end, (uint64_t)p.max_tok);
        row0 += sum;
        const uint64_t kv = held + (r1 - r0);
        const uint64_t before = min((held + ps - 1) >> sh, (uint64_t)p.table_stride);
        const uint64_t need = min((kv + ps - 1) >> sh, (uint64_t)p.table_stride) - before;
        const uint64_t first = page0 + scan_wg(need, ws, &sum) - need;
        const uint64_t pages = sum;
        l_row[tid] = r0;
        l_rows[tid] = r1 - r0;
        l_held[tid] = (uint32_t)held;
        l_before[tid] = (uint32_t)before;
        l_page[tid] = first - page0;
        if (in) {
            // rows without a slot: those cut off, those behind the table's row, and in the page
            // begun before; the new pages' are counted where the pages are dealt
            const uint64_t end_at = (before + need) << sh, begun = min(kv, before << sh);
            lost += add - (r1 - r0) + (kv - max(min(kv, end_at), held));
            if (begun > held) lost += lost_in(p.table[(uint64_t)s * p.table_stride + before - 1], held, begun, sh);
            p.q_start[s] = r0;
            p.kv_len[s] = sat32(kv);
        }
        __syncthreads();
        for (uint64_t i = tid; i < pages; i += PLAN_T) {
            const uint32_t q = owner(l_page, nb, i);
            const uint64_t at = page0 + i, pg = l_before[q] + (i - l_page[q]);
            const uint32_t g = at < p.n_free ? p.free_pages[at] : FLH_KV_NONE;
            p.table[(uint64_t)(base + q) * p.table_stride + pg] = g;
            const uint64_t held = l_held[q];
            lost += lost_in(g, max(held, pg << sh), min(held + l_rows[q], (pg + 1) << sh), sh);
        }
        if (rows_too) {
            const uint32_t e = (uint32_t)min(row0, (uint64_t)p.max_tok);
            for (uint32_t i = l_row[0] + tid; i < e; i += PLAN_T) {
                const uint32_t q = owner(l_row, nb, i);
                const uint64_t at = (uint64_t)l_held[q] + (i - l_row[q]), pg = at >> sh;
                uint32_t g = FLH_KV_NONE;
                if (pg < l_before[q]) g = p.table[(uint64_t)(base + q) * p.table_stride + pg];
                else if (pg < p.table_stride) {
                    const uint64_t f = page0 + l_page[q] + (pg - l_before[q]);
                    if (f < p.n_free) g = p.free_pages[f];
                }
                p.slot[i] = slot_of(g, (uint32_t)at, sh);
                if (p.pos) p.pos[i] = (int32_t)(uint32_t)at;
            }
        }
        page0 += pages;
        __syncthreads();                                          // the tables in LDS are the next batch's
    }
    const uint32_t rows = (uint32_t)min(row0, (uint64_t)p.max_tok);
    if (rows_too)
        for (uint32_t i = rows + tid; i < p.max_tok; i += PLAN_T) {
            p.slot[i] = FLH_KV_NONE;
            if (p.pos) p.pos[i] = 0;
        }
    uint64_t all;
    (void)scan_wg(lost, ws, &all);
    if (tid == 0) {
        p.q_start[p.n_seq] = rows;
        *p.taken = sat32(page0);
        if (p.info) {
            p.info[0] = rows;
            p.info[1] = sat32(all);
        }
    }
}

// Slots and positions of many rows, a thread each, from the finished table.
__global__ __launch_bounds__(256) void k_kv_slots(flh_kv_plan_p p, uint32_t sh) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= p.max_tok) return;
    if (i >= p.q_start[p.n_seq]) {
        p.slot[i] = FLH_KV_NONE;
        if (p.pos) p.pos[i] = 0;
        return;
    }
    const uint32_t s = owner(p.q_start, p.n_seq, i);
    const uint32_t r0 = p.q_start[s], n = p.q_start[s + 1] - r0;
    const uint64_t at = (uint64_t)(p.kv_len[s] - n) + (i - r0), pg = at >> sh;
    const uint32_t g = pg < p.table_stride ? p.table[(uint64_t)s * p.table_stride + pg] : FLH_KV_NONE;
    p.slot[i] = slot_of(g, (uint32_t)at, sh);
    if (p.pos) p.pos[i] = (int32_t)(uint32_t)at;
}

int launch_kv_plan(const flh_kv_plan_p & p, hipStream_t s) {
    constexpr uint32_t PLAN_ROWS = 6144;
    const uint32_t sh = (uint32_t)__builtin_ctz(p.page_size);
    const bool one = p.max_tok <= PLAN_ROWS;
    hipLaunchKernelGGL(k_kv_plan, dim3(1), dim3(PLAN_T), 0, s, p, sh, one ? 1 : 0);
    if (int rc = hip_check(hipGetLastError(), "k_kv_plan launch")) return rc;
    if (one) return FLH_OK;
    hipLaunchKernelGGL(k_kv_slots, dim3((uint32_t)(((uint64_t)p.max_tok + 255) / 256)), dim3(256), 0, s, p, sh);
    return hip_check(hipGetLastError(), "k_kv_slots launch");
}

// ------------------------------------------------------------------- rope --
// cos and sin of pair `t` at its position: turn = pos * frac mod 2^64 is the
// angle as a fraction of a turn, off by at most |pos| * 2^-65 (frac is rounded once; below
// 2^-34 for every 32-bit position).  The nearest quarter turn comes off in integers, so the
// rest, at most an eighth of a turn, keeps 24 bits as a float however small it is: the sines of
// slow pairs at near positions are as good as their cosines.
__device__ __forceinline__ void rope_cs(const RopePair & t, const int32_t * pos, uint32_t pos_stride, uint32_t tok,
                                        float & c, float & s) {
    const uint64_t turn = (uint64_t)(int64_t)pos[(size_t)t.axis * pos_stride + tok] * t.frac;
    const uint32_t q = (uint32_t)((turn + (1ull << 61)) >> 62);
    const float r = (float)(int64_t)(turn - ((uint64_t)q << 62)) * 0x1p-63f;   // half turns
    float s0, c0;
    sincospif(r, &s0, &c0);
    const float a = q & 1 ? s0 : c0, b = q & 1 ? c0 : s0;
    c = (q + 1) & 2 ? -a : a;
    s = q & 2 ? -b : b;
}

template <typename T, int N> struct alignas(sizeof(T) * N) Vec { T v[N]; };
template <int N, typename T> __device__ __forceinline__ Vec<T, N> ld_vec(const T * p) { return *(const Vec<T, N> *)p; }
template <int N, typename T> __device__ __forceinline__ void st_vec(T * p, const float * y) {
    Vec<T, N> o;
#pragma unroll
    for (int i = 0; i < N; ++i) o.v[i] = (T)y[i];
    *(Vec<T, N> *)p = o;
}

// Token tok0 + blockIdx.x; its heads of q and then k are cut into units of N pairs or
// 2N other elements (the last may have N), its heads of v into units of N, and
// the workgroups of blockIdx.y share them.  Nothing is used twice but the
// angles: a workgroup makes each once, behind the loads of its threads' first
// units, and every head reads them from LDS.  Bytes bound it: 4999 tokens of 32 + 8 heads
// of 128 with values in bf16 take 27 us (4.5 TB/s; a large copy reaches 5.1), 1000 tokens
// of 16 + 16 heads of 192 in fp32 11.0 us (5.0 TB/s), one token 7.4 us, a launch and
// its chain of loads (2.8 us on the device).  One thread per pair with its own angle took 64.5, 23.6 and 7.3;
// two units in flight instead of one 30.6.
struct RopeUnits {
    uint32_t pu, u, n, step_h, step_e;     // a head's pair units and all its units, their number, and a step in (head, unit)
};
constexpr uint32_t ROPE_T = 256;
template <typename AT, typename CT, int N>
__global__ __launch_bounds__(ROPE_T) void k_rope(RopeArgs a, RopeUnits ru) {
    __shared__ float2 cs[512];
    const uint32_t tok = a.tok0 + blockIdx.x, nk = a.kc ? a.n_kv : 0, P = a.rot ? a.n_rot / 2 : 0;
    const uint32_t first = blockIdx.y * ROPE_T + threadIdx.x, step = gridDim.y * ROPE_T;
    const uint32_t slot = nk ? a.slot[tok] : 0;
    const bool live = nk && slot < a.n_slot;
    const uint64_t page = slot >> a.sh, off = slot & ((1u << a.sh) - 1u);
    const AT * q = (const AT *)a.q + tok * a.q_tok, * k = (const AT *)a.k + tok * a.k_tok;
    AT * qo = (AT *)a.qo + tok * a.qo_tok;
    CT * kc = (CT *)a.kc + page * a.kc_page + off * a.kc_tok;

    uint32_t h = first / ru.u, e = first - h * ru.u;
    for (uint32_t at = first, round = 0; round == 0 || at - threadIdx.x < ru.n; ++round) {
        Vec<AT, N> x, w;
        uint32_t i0, j0;                   // where the unit's two vectors are in the head
        bool two = true;
        const bool on = at < ru.n && (h < a.n_head || live), isq = h < a.n_head;
        if (e < ru.pu) {
            i0 = a.first + (a.halves ? e * N : e * 2 * N);
            j0 = i0 + (a.halves ? P : N);
        } else {
            const uint32_t r = (e - ru.pu) * 2 * N;              // among the elements that are not turned
            i0 = r < a.first || !P ? r : r + 2 * P;
            j0 = r + N < a.first || !P ? r + N : r + N + 2 * P;
            two = r + N < a.d - 2 * P;
        }
        if (on) {
            const AT * src = isq ? q + h * a.q_head : k + (h - a.n_head) * a.k_head;
            x = ld_vec<N>(src + i0);
            if (two) w = ld_vec<N>(src + j0);
        }
        if (round == 0) {
            for (uint32_t i = threadIdx.x; i < P; i += ROPE_T)
                rope_cs(a.rot[i], a.pos, a.pos_stride, tok, cs[i].x, cs[i].y);
            __syncthreads();
        }
        if (on) {
            float y[N], z[N];
            if (e < ru.pu) {
                const float2 * t = cs + e * N;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float c = t[i].x, s = t[i].y;
                    // halves: pair i is (x[i], w[i]); pairs: the 2N elements x, w one after the other
                    const float v = (float)(a.halves ? x.v[i] : 2 * i < N ? x.v[2 * i % N] : w.v[2 * i % N]);
                    const float u = (float)(a.halves ? w.v[i] : 2 * i + 1 < N ? x.v[(2 * i + 1) % N] : w.v[(2 * i + 1) % N]);
                    const float ya = v * c - u * s, yb = v * s + u * c;
                    if (a.halves) {
                        y[i] = ya;
                        z[i] = yb;
                    } else if constexpr (N == 1) {
                        y[0] = ya;
                        z[0] = yb;
                    } else if (2 * i < N) {
                        y[2 * i % N] = ya;
                        y[(2 * i + 1) % N] = yb;
                    } else {
                        z[2 * i % N] = ya;
                        z[(2 * i + 1) % N] = yb;
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    y[i] = (float)x.v[i];
                    z[i] = (float)w.v[i];
                }
            }
            if (isq) {
                AT * d = qo + h * a.qo_head;
                st_vec<N>(d + i0, y);
                if (two) st_vec<N>(d + j0, z);
            } else {
                CT * d = kc + (h - a.n_head) * a.kc_head;
                st_vec<N>(d + i0, y);
                if (two) st_vec<N>(d + j0, z);
            }
        }
        at += step; h += ru.step_h; e += ru.step_e;
        if (e >= ru.u) { e -= ru.u; ++h; }
    }
    if (!live) return;
    const uint32_t vu = a.dv / N;
    const AT * v = (const AT *)a.v + tok * a.v_tok;
    CT * vc = (CT *)a.vc + page * a.vc_page + off * a.vc_tok;
    for (uint32_t at = first; at < nk * vu; at += step) {
        const uint32_t hv = at / vu, i = (at - hv * vu) * N;
        const Vec<AT, N> x = ld_vec<N>(v + hv * a.v_head + i);
        float y[N];
#pragma unroll
        for (int j = 0; j < N; ++j) y[j] = (float)x.v[j];
        st_vec<N>(vc + hv * a.vc_head + i, y);
    }
}

template <typename AT, typename CT, int N>
static int rope_n(RopeArgs a, hipStream_t s) {
    const uint32_t P = a.rot ? a.n_rot / 2 : 0, nk = a.kc ? a.n_kv : 0, rest = a.d - 2 * P;
    RopeUnits ru;
    ru.pu = P / N;
    ru.u = ru.pu + (rest + 2 * N - 1) / (2 * N);
    ru.n = ru.u * (a.n_head + nk);
    const uint32_t most = (uint32_t)((std::max<uint64_t>(ru.n, nk * a.dv / N) + ROPE_T - 1) / ROPE_T);
    // Few tokens: workgroups share a token's units.  us so / with one workgroup a token, 128 + 8
    // heads of 192 in bf16: 4 tokens 7.1 / 7.7, 64 6.7 / 8.1, 256 8.1 / 9.5, 512 12.7 / 12.8; 32 + 8 heads of 128 in
    // fp32 7.3 / 7.7, 7.0 / 6.8, 6.7 / 7.1, 6.8 / 7.0; one token 7.3 to 7.5 either way.
    const uint32_t parts = std::max(1u, std::min(most, 512 / a.n_tok));
    ru.step_h = parts * ROPE_T / ru.u;
    ru.step_e = parts * ROPE_T % ru.u;
    constexpr uint32_t MOST_TOK = 1u << 22;            // of a launch: its threads are counted in 32 bits
    for (uint64_t t = 0; t < a.n_tok; t += MOST_TOK) {
        a.tok0 = (uint32_t)t;
        hipLaunchKernelGGL((k_rope<AT, CT, N>), dim3(std::min(a.n_tok - a.tok0, MOST_TOK), parts), dim3(ROPE_T), 0, s, a, ru);
        if (int rc = hip_check(hipGetLastError(), "k_rope launch")) return rc;
    }
    return FLH_OK;
}
// whether every head of every token allows units of n elements
static bool rope_fits(const RopeArgs & a, uint32_t el, uint32_t n) {
    auto fit = [n](const void * p, uint32_t e, uint64_t tok, uint64_t head) {
        return (uintptr_t)p % (e * n) == 0 && tok % n == 0 && head % n == 0;
    };
    const uint32_t P = a.rot ? a.n_rot / 2 : 0;
    if (P % n || (P && a.first % n) || a.d % n) return false;
    if (a.n_head && !(fit(a.q, el, a.q_tok, a.q_head) && fit(a.qo, el, a.qo_tok, a.qo_head))) return false;
    return !a.kc || (fit(a.k, el, a.k_tok, a.k_head) && fit(a.v, el, a.v_tok, a.v_head) && a.dv % n == 0 &&
                     fit(a.kc, 2, a.kc_page | a.kc_tok, a.kc_head) && fit(a.vc, 2, a.vc_page | a.vc_tok, a.vc_head));
}
// Units of 16 bytes where alignment allows them, else single elements.
template <typename AT, typename CT>
static int rope_c(const RopeArgs & a, hipStream_t s) {
    constexpr int N = 16 / sizeof(AT);
    if (rope_fits(a, sizeof(AT), N)) return rope_n<AT, CT, N>(a, s);
    return rope_n<AT, CT, 1>(a, s);
}
template <typename AT>
static int rope_go(const RopeArgs & a, uint32_t cdt, hipStream_t s) {
    return cdt == FLH_DT_BF16 ? rope_c<AT, __bf16>(a, s) : rope_c<AT, _Float16>(a, s);
}
int launch_rope(const RopeArgs & a, uint32_t dtype, uint32_t cache_dtype, hipStream_t s) {
    if (dtype == FLH_DT_F32) return rope_go<float>(a, cache_dtype, s);
    if (dtype == FLH_DT_F16) return rope_go<_Float16>(a, cache_dtype, s);
    return rope_go<__bf16>(a, cache_dtype, s);
}

}  // namespace flh
