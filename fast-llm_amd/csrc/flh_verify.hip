// flh_verify.hip -- verification of drafted tokens: which rows of a request's tree stand
// against the target's distribution, and the token behind them.
//
// Let p be softmax(inv_temp * target) and q softmax(inv_temp * draft) of a row, and x_0, x_1, ..
// the tokens of its children, drawn from q.  Child i stands where u q(x_i) < p_i(x_i), with p_0 = p
// and, as each child that does not stand takes its share away, p_(i+1) = max(p_i - q, 0) over its sum.  No
// such distribution is ever stored: p_i = max(p - t_i q, 0) / n_i with t_0 = 0, n_0 = 1 and
//     t_(i+1) = t_i + n_i,    n_i = sum over the vocabulary of max(p - t_i q, 0),
// for p_i - q is (p - t_i q - n_i q) / n_i where p > t_i q, and not positive elsewhere.  So a
// row of k children costs k numbers: n_1 .. n_(k-1) for the tests, a launch each over the rows that
// have so many, and n_k on the way of drawing the token behind the last row.  Without a
// draft's distribution q is 1 at the token itself: p_i is p without the tokens before.
//
// Launches: sums of every row's chunks (bytes bound it); n_i (only with several
// children a row); the walk and the draw.  A random number may lie next to
// the border of two of 10^5 tokens, so weights, sums and borders are in 64 bits: with the
// exponential below an element costs about 20 instructions, as much time as its bytes in fp32.
#include "flh_common.h"
#include "flh_internal.h"
#include "flh_status.h"
#include <float.h>

namespace flh {

constexpr uint32_t VER_T = 256, VER_N = 16, VER_CH = VER_T * VER_N;   // threads, elements a thread, of a chunk
constexpr uint32_t VER_ROWS = 256;                                    // of a request that are looked at
constexpr uint32_t NO_ROW = 0xFFFFFFFFu;

// A chunk's largest logit, where it first is (greedy requests), and the sum of
// exp((x - m) inv_temp).
struct VerPart {
    double z;
    float m;
    uint32_t at;
};
struct VerArgs {
    flh_verify_p p;
    VerPart * tp, * dp;                 // [n_tok][nc]
    double * rest;                      // [max_child - 1][n_tok][nc]: n_1 ..
    double * left;                      // [n_seq][nc]
    uint32_t * done;                    // [n_seq]
    uint32_t nc, rounds, share;         // chunks of a row; launches of k_verify_rest; workgroups of a request's draw
};

// e^y for y <= 0 (0 below -1000, and for what is no number): y = k ln 2 + f, |f| <= ln 2 / 2, the series of
// e^f up to f^11 / 11! (6e-15 are left out).
__device__ __forceinline__ double exp_down(double y) {
    y = fmax(y, -1000.0);
    const double k = rint(y * 1.4426950408889634074);
    double f = fma(-k, 0x1.62e42fefa39efp-1, y);                      // ln 2 in two parts
    f = fma(-k, 0x1.abc9e3b39803fp-56, f);
    double e = 1.0 / 39916800;
    e = fma(e, f, 1.0 / 3628800);
    e = fma(e, f, 1.0 / 362880);
    e = fma(e, f, 1.0 / 40320);
    e = fma(e, f, 1.0 / 5040);
    e = fma(e, f, 1.0 / 720);
    e = fma(e, f, 1.0 / 120);
    e = fma(e, f, 1.0 / 24);
    e = fma(e, f, 1.0 / 6);
    e = fma(e, f, 0.5);
    e = fma(e, f, 1.0);
    e = fma(e, f, 1.0);
    return ldexp(e, (int)k);
}
// a logit: what is no number counts as -infinity, infinity as the largest number
__device__ __forceinline__ float logit(float x) { return x == x ? fminf(x, FLT_MAX) : -INFINITY; }
// exp((x - m) it) where m is the largest x (or -infinity, where no x is more)
__device__ __forceinline__ double weight(float x, float m, double it) {
    return exp_down(((double)x - (m == -INFINITY ? 0.0 : (double)m)) * it);
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    return v;
}

// Elements [at, at + n) of a row of v (n = 4 or 8 of 16 bytes; -infinity behind the row's end).
template <typename T, int N> __device__ __forceinline__ void load_logits(const T * row, uint32_t at, uint32_t v, float (&x)[N]) {
    struct alignas(sizeof(T)) V { T v[N]; };
    if (at + N <= v) {
        V t;
        __builtin_memcpy(&t, row + at, sizeof t);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = logit((float)t.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = at + i < v ? logit((float)row[at + i]) : -INFINITY;
    }
}
// A thread's elements of a chunk: pieces of 16 bytes, the workgroup's side by side
template <typename T> __device__ __forceinline__ void load_chunk(const T * row, uint32_t c0, uint32_t v, float (&x)[VER_N]) {
    constexpr int N = 16 / sizeof(T);
#pragma unroll
    for (int j = 0; j < (int)VER_N / N; ++j) {
        float y[N];
        load_logits<T, N>(row, c0 + (j * VER_T + threadIdx.x) * N, v, y);
#pragma unroll
        for (int i = 0; i < N; ++i) x[j * N + i] = y[i];
    }
}
// where element i of load_chunk's is
template <typename T> __device__ __forceinline__ uint32_t chunk_at(uint32_t c0, int i) {
    constexpr int N = 16 / sizeof(T);
    return c0 + (i / N * VER_T + threadIdx.x) * N + i % N;
}
// Sum over the workgroup, the same in every thread (sm: 4 values; waves are added in order)
__device__ __forceinline__ double wg_sum(double v, double * sm) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = v;
    __syncthreads();
    return sm[0] + sm[1] + sm[2] + sm[3];
}

__device__ __forceinline__ double inv_temp_of(const flh_verify_p & p, uint32_t s) {
    const float it = p.inv_temp ? p.inv_temp[s] : 1.f;
    return it >= 0.f ? (double)it : 0.0;                              // (infinity: greedy)
}
// the request of a row, NO_ROW for a row of none
__device__ __forceinline__ uint32_t request_of(const flh_verify_p & p, uint32_t row) {
    if (row < p.q_start[0] || row >= p.q_start[p.n_seq]) return NO_ROW;
    uint32_t lo = 0, n = p.n_seq;
    while (n > 1) {
        const uint32_t h = n >> 1;
        if (p.q_start[lo + h] <= row) { lo += h; n -= h; }
        else n = h;
    }
    return lo;
}
__device__ __forceinline__ uint32_t rows_of(const flh_verify_p & p, uint32_t s, uint32_t & r0) {
    r0 = min(p.q_start[s], p.n_tok);
    const uint32_t end = min(p.q_start[s + 1], p.n_tok);
    return end > r0 ? min(end - r0, VER_ROWS) : 0u;
}
// the row that row i of a request hangs on (NO_ROW: none)
__device__ __forceinline__ uint32_t parent_of(const flh_verify_p & p, uint32_t r0, uint32_t i) {
    const uint32_t x = p.parent ? (uint32_t)p.parent[r0 + i] : i - 1;
    return x < i ? x : NO_ROW;
}
// children of row i of a request of n rows (every thread of the workgroup the same)
__device__ __forceinline__ uint32_t children(const flh_verify_p & p, uint32_t r0, uint32_t n, uint32_t i) {
    if (!p.parent) return i + 1 < n;
    uint32_t k = 0;
    for (uint32_t j = i + 1; j < n; j += VER_T) k += __syncthreads_count(j + threadIdx.x < n && parent_of(p, r0, min(j + threadIdx.x, n - 1)) == i);
    return min(k, p.max_child);
}

// ------------------------------------------------------------- the rows' sums --
// Workgroup (row, chunk) of the target (y = 0) or of the draft (1: rows with children).
template <typename T> __global__ __launch_bounds__(VER_T) void k_verify_sums(VerArgs a) {
    __shared__ float sm_m[4];
    __shared__ double sm_z[4];
    __shared__ uint32_t sm_at[4];
    const flh_verify_p & p = a.p;
    const uint32_t row = blockIdx.x / a.nc, c = blockIdx.x % a.nc, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool draft = blockIdx.y != 0;
    if (blockIdx.x == 0 && draft)
        for (uint32_t i = threadIdx.x; i < p.n_seq; i += VER_T) a.done[i] = 0;
    const uint32_t s = request_of(p, row);
    if (s == NO_ROW) return;
    const double it = inv_temp_of(p, s);
    const bool greedy = isinf(it);
    if (draft) {
        uint32_t r0;
        const uint32_t n = rows_of(p, s, r0);
        if (greedy || row - r0 >= n || children(p, r0, n, row - r0) == 0) return;
    }
    float x[VER_N], m = -INFINITY;
    load_chunk<T>(draft ? (const T *)p.draft + row * p.d_row : (const T *)p.target + row * p.t_row, c * VER_CH, p.vocab, x);
#pragma unroll
    for (int i = 0; i < (int)VER_N; ++i) m = fmaxf(m, x[i]);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
    double z = 0;
    uint32_t at = NO_ROW;
    if (greedy) {
#pragma unroll
        for (int i = (int)VER_N - 1; i >= 0; --i) at = x[i] == m && m > -INFINITY ? min(at, chunk_at<T>(c * VER_CH, i)) : at;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) at = min(at, (uint32_t)__shfl_xor((int)at, d));
    } else {
#pragma unroll
        for (int i = 0; i < (int)VER_N; ++i) z += weight(x[i], m, it);
        z = wave_sum(z);
    }
    if (lane == 0) {
        sm_m[wave] = m;
        sm_z[wave] = z;
        sm_at[wave] = at;
    }
    __syncthreads();
    if (threadIdx.x) return;
    VerPart o{0, fmaxf(fmaxf(sm_m[0], sm_m[1]), fmaxf(sm_m[2], sm_m[3])), NO_ROW};
    for (int w = 0; w < 4; ++w) {
        if (sm_m[w] == o.m) o.at = min(o.at, sm_at[w]);
        o.z += sm_z[w] * weight(sm_m[w], o.m, greedy ? 1.0 : it);
    }
    (draft ? a.dp : a.tp)[(uint64_t)row * a.nc + c] = o;
}

// A row's largest logit and sum from its chunks', by the lanes of a group of G in step; and
// where the largest first is
struct VerRow {
    float m;
    double z;
    uint32_t at;
};
template <int G> __device__ __forceinline__ VerRow merge_row(const VerPart * part, uint32_t nc, double it) {
    const uint32_t l = threadIdx.x % G;
    VerRow r{-INFINITY, 0.0, NO_ROW};
    for (uint32_t c = l; c < nc; c += G) r.m = fmaxf(r.m, part[c].m);
#pragma unroll
    for (int d = 1; d < G; d <<= 1) r.m = fmaxf(r.m, __shfl_xor(r.m, d));
    for (uint32_t c = l; c < nc; c += G) {
        const VerPart q = part[c];
        if (q.m == r.m) r.at = min(r.at, q.at);
        r.z += q.z * weight(q.m, r.m, it);
    }
#pragma unroll
    for (int d = 1; d < G; d <<= 1) {
        r.z += __shfl_xor(r.z, d);
        r.at = min(r.at, (uint32_t)__shfl_xor((int)r.at, d));
    }
    return r;
}
// n_j of a row (j >= 1), and t_i = 1 + n_1 + .. + n_(i-1) (i >= 1), by the lanes of a group of G in step
template <int G> __device__ __forceinline__ double rest_of(const VerArgs & a, uint32_t row, uint32_t j) {
    const double * r = a.rest + ((uint64_t)(j - 1) * a.p.n_tok + row) * a.nc;
    double n = 0;
    for (uint32_t c = threadIdx.x % G; c < a.nc; c += G) n += r[c];
#pragma unroll
    for (int d = 1; d < G; d <<= 1) n += __shfl_xor(n, d);
    return n;
}
template <int G> __device__ __forceinline__ double taken_of(const VerArgs & a, uint32_t row, uint32_t i) {
    double t = 1.0;
    for (uint32_t j = 1; j < i; ++j) t += rest_of<G>(a, row, j);
    return t;
}

// n_i, i = `round`, of the rows with more than i children: workgroup (row, chunk).
template <typename T> __global__ __launch_bounds__(VER_T) void k_verify_rest(VerArgs a, uint32_t round) {
    __shared__ double sm[4];
    const flh_verify_p & p = a.p;
    const uint32_t row = blockIdx.x / a.nc, c = blockIdx.x % a.nc;
    const uint32_t s = request_of(p, row);
    if (s == NO_ROW) return;
    const double it = inv_temp_of(p, s);
    uint32_t r0;
    const uint32_t n = rows_of(p, s, r0);
    if (isinf(it) || row - r0 >= n || children(p, r0, n, row - r0) <= round) return;
    float x[VER_N], y[VER_N];
    load_chunk<T>((const T *)p.target + row * p.t_row, c * VER_CH, p.vocab, x);
    load_chunk<T>((const T *)p.draft + row * p.d_row, c * VER_CH, p.vocab, y);
    const double t = taken_of<64>(a, row, round);
    const VerRow tr = merge_row<64>(a.tp + (uint64_t)row * a.nc, a.nc, it), dr = merge_row<64>(a.dp + (uint64_t)row * a.nc, a.nc, it);
    const double fp = tr.z > 0 ? 1.0 / tr.z : 0.0, fq = dr.z > 0 ? t / dr.z : 0.0;
    double sum = 0;
#pragma unroll
    for (int i = 0; i < (int)VER_N; ++i) sum += fmax(weight(x[i], tr.m, it) * fp - weight(y[i], dr.m, it) * fq, 0.0);
    sum = wg_sum(sum, sm);
    if (threadIdx.x == 0) a.rest[((uint64_t)(round - 1) * p.n_tok + row) * a.nc + c] = sum;
}

// -------------------------------------------------------- the walk and the draw --
struct VerWalk {
    double tz[VER_ROWS], dz[VER_ROWS], pc[VER_ROWS];                  // sums of rows; p of rows' tokens
    double t[VER_ROWS], n[VER_ROWS];                                  // what rows' tests are against
    uint32_t at[VER_ROWS];                                            // where rows' largest are (greedy)
    float tm[VER_ROWS], dm[VER_ROWS];
    uint32_t up[VER_ROWS], best[VER_ROWS];                            // parents; first child that stands
    uint8_t rank[VER_ROWS], kids[VER_ROWS];                           // among its siblings (255: behind max_child)
    uint32_t end, len, k;                                             // the last row, the path's rows, children looked at
};

// The row's weights of a chunk's elements, e(x) or max(p - t q, 0).
struct VerLeft {
    double it, fp, fq;
    float tm, dm;
    __device__ __forceinline__ double of(float x, float y) const { return fmax(weight(x, tm, it) * fp - weight(y, dm, it) * fq, 0.0); }
};

template <typename T> __global__ __launch_bounds__(VER_T) void k_verify_next(VerArgs a) {
    __shared__ VerWalk w;
    __shared__ double sm[4], sums[1024];
    __shared__ uint32_t sm_last, sm_pick, gone[VER_ROWS], n_gone;
    const flh_verify_p & p = a.p;
    const uint32_t s = blockIdx.x / a.share, part = blockIdx.x % a.share, tid = threadIdx.x;
    const double it = inv_temp_of(p, s);
    const bool greedy = isinf(it);
    uint32_t r0;
    const uint32_t n = rows_of(p, s, r0);
    const uint64_t out = (uint64_t)s * p.path_stride;
    if (n == 0) {
        if (part) return;
        for (uint32_t j = tid; j < p.path_stride; j += VER_T) {
            p.path[out + j] = FLH_KV_NONE;
            if (p.logp) p.logp[out + j] = 0.f;
        }
        if (tid == 0) {
            p.n_path[s] = 0;
            p.next[s] = FLH_KV_NONE;
            if (p.len) p.len[s] = p.kv_len[s];
        }
        return;
    }
    // ---- the rows' parents, and their sums where they have children
    for (uint32_t i = tid; i < n; i += VER_T) {
        w.up[i] = i ? parent_of(p, r0, i) : NO_ROW;
        w.best[i] = NO_ROW;
        w.kids[i] = 0;
    }
    __syncthreads();
    for (uint32_t i = tid; i < n; i += VER_T) {
        const uint32_t u = w.up[i];
        uint32_t k = 0;
        if (u != NO_ROW) {
            w.kids[u] = 1;                                            // (others write the same)
            for (uint32_t j = u + 1; j < i; ++j) k += w.up[j] == u;
        }
        w.rank[i] = u == NO_ROW || k >= p.max_child ? 255 : (uint8_t)k;
    }
    __syncthreads();
    for (uint32_t i0 = 0; i0 < n; i0 += VER_T / 32) {                 // 32 lanes a row
        const uint32_t i = i0 + tid / 32;
        const bool on = i < n && (w.kids[min(i, n - 1)] || i == 0);
        const uint64_t row = r0 + min(i, n - 1);
        if (!__ballot(on)) continue;
        const VerRow t = merge_row<32>(a.tp + row * a.nc, on ? a.nc : 0, greedy ? 1.0 : it);
        const VerRow d = merge_row<32>(a.dp + row * a.nc, on && p.draft && !greedy ? a.nc : 0, it);
        if (on && tid % 32 == 0) {
            w.tm[i] = t.m;
            w.at[i] = t.at;
            w.tz[i] = t.z;
            w.dm[i] = d.m;
            w.dz[i] = d.z;
        }
    }
    __syncthreads();
    // ---- which rows stand against their parent's distribution
    for (uint32_t i = tid; i < n; i += VER_T) {
        const uint32_t u = w.up[i];
        double pc = 0;
        if (u != NO_ROW) {
            const uint32_t x = p.token[r0 + i];
            if (x < p.vocab) {
                if (greedy) pc = w.at[u] == x ? 1.0 : 0.0;
                else if (w.tz[u] > 0) pc = weight(logit((float)((const T *)p.target)[(r0 + u) * p.t_row + x]), w.tm[u], it) / w.tz[u];
            }
        }
        w.pc[i] = pc;
    }
    if (a.rounds && !greedy)                                          // (rows of one child each: t is 0, n is 1)
        for (uint32_t i0 = 0; i0 < n; i0 += VER_T / 32) {
            const uint32_t i = min(i0 + tid / 32, n - 1), k = w.rank[i] == 255 ? 0 : w.rank[i];
            double t = 0, m = 1;
            for (uint32_t j = 1; __ballot(j <= k); ++j) {             // (the halves of a wave together)
                const double r = rest_of<32>(a, r0 + (j <= k ? w.up[i] : 0), j);
                t = j <= k ? t + m : t;
                m = j <= k ? r : m;
            }
            w.t[i] = t;
            w.n[i] = m;
        }
    __syncthreads();
    for (uint32_t i = tid; i < n; i += VER_T) {
        const uint32_t u = w.up[i], k = w.rank[i];
        if (u == NO_ROW || k == 255) continue;
        const uint32_t x = p.token[r0 + i];
        const double pc = w.pc[i], uu = p.u_accept[r0 + i];
        bool ok;
        if (greedy) ok = pc > 0;
        else if (p.draft) {
            double qc = 0, t = 0, nn = 1;
            if (x < p.vocab && w.dz[u] > 0)
                qc = weight(logit((float)((const T *)p.draft)[(r0 + u) * p.d_row + x]), w.dm[u], it) / w.dz[u];
            if (k) {
                t = w.t[i];
                nn = w.n[i];
            }
            ok = uu * qc * nn < fmax(pc - t * qc, 0.0);
        } else {
            double took = 0;
            bool twice = false;
            for (uint32_t j = u + 1; j < i; ++j) {
                if (w.up[j] != u) continue;
                const uint32_t y = p.token[r0 + j];
                twice = twice || y == x;
                bool again = false;
                for (uint32_t l = u + 1; l < j; ++l) again = again || (w.up[l] == u && p.token[r0 + l] == y);
                if (!again) took += w.pc[j];
            }
            ok = !twice && uu * (1.0 - took) < pc;
        }
        if (ok) atomicMin(&w.best[u], i);
    }
    __syncthreads();
    // ---- the path: from row 0 on, the first child that stands
    if (tid == 0) {
        uint32_t cur = 0, len = 1;
        while (len < p.path_stride && w.best[cur] != NO_ROW) {
            cur = w.best[cur];
            ++len;
        }
        w.end = cur;
        w.len = len;
        // a path cut off ends as at a row without children
        w.k = w.best[cur] == NO_ROW;
        n_gone = 0;
    }
    __syncthreads();
    const uint32_t end = w.end;
    const uint64_t row = r0 + end;
    if (w.k) {                                                        // its children, and their tokens
        uint32_t k = 0;
        for (uint32_t j0 = end + 1; j0 < n; j0 += VER_T) {
            const uint32_t j = j0 + tid;
            const bool mine = j < n && w.up[min(j, n - 1)] == end && w.rank[min(j, n - 1)] != 255;
            k += __syncthreads_count(mine);
            if (mine) gone[atomicAdd(&n_gone, 1u)] = p.token[r0 + j];
        }
        if (tid == 0) w.k = k;
        __syncthreads();
    }
    const uint32_t k = greedy ? 0 : w.k;
    const bool both = p.draft && k;                                   // what is left of p takes a pass over the row
    if (part && !both) return;
    // (a leaf's sums are still to be merged)
    VerLeft f{it, 1.0, 0.0, -INFINITY, -INFINITY};
    VerRow tr = merge_row<64>(a.tp + row * a.nc, a.nc, greedy ? 1.0 : it);
    f.tm = tr.m;
    const T * xr = (const T *)p.target + row * p.t_row;
    const T * yr = both ? (const T *)p.draft + row * p.d_row : nullptr;
    bool plain = !both;
    if (both) {
        const VerRow dr = merge_row<64>(a.dp + row * a.nc, a.nc, it);
        const double t = taken_of<64>(a, (uint32_t)row, k);
        f.dm = dr.m;
        f.fp = tr.z > 0 ? 1.0 / tr.z : 0.0;
        f.fq = dr.z > 0 ? t / dr.z : 0.0;
        float x[VER_N], y[VER_N];
        load_chunk<T>(xr, part * VER_CH, p.vocab, x);
        load_chunk<T>(yr, part * VER_CH, p.vocab, y);
        double sum = 0;
#pragma unroll
        for (int i = 0; i < (int)VER_N; ++i) sum += f.of(x[i], y[i]);
        sum = wg_sum(sum, sm);
        // the last workgroup of the request draws
        if (tid == 0) {
            __hip_atomic_store(a.left + (uint64_t)s * a.nc + part, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __threadfence();
            sm_last = atomicAdd(a.done + s, 1u) == a.nc - 1;
            __threadfence();
        }
        __syncthreads();
        if (!sm_last) return;
        for (uint32_t c = tid; c < a.nc; c += VER_T)
            sums[c] = __hip_atomic_load(a.left + (uint64_t)s * a.nc + c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        double all = 0;
        __syncthreads();
        for (uint32_t c = tid; c < a.nc; c += VER_T) all += sums[c];
        if (!(wg_sum(all, sm) > 0)) {                                 // nothing is left of p: p itself
            plain = true;
            f.fp = 1.0;
            f.fq = 0.0;
        }
    }
    uint32_t next = FLH_KV_NONE;
    uint32_t cut = plain && !p.draft && k ? n_gone : 0;               // tokens that are taken out
    if (greedy) next = tr.m == -INFINITY ? FLH_KV_NONE : tr.at;
    else if (tr.m != -INFINITY) {
        // a chunk's weights in the order of the tokens, 16 a thread
        double e[VER_N];
        auto chunk = [&](uint32_t c) {
            const uint32_t at = c * VER_CH + tid * VER_N;
            float x[VER_N], y[VER_N];
            load_logits<T, (int)VER_N>(xr, at, p.vocab, x);
            if (!plain) load_logits<T, (int)VER_N>(yr, at, p.vocab, y);
#pragma unroll
            for (int i = 0; i < (int)VER_N; ++i) e[i] = plain ? weight(x[i], f.tm, it) : f.of(x[i], y[i]);
            for (uint32_t g = 0; g < cut; ++g) {
                const uint32_t d = gone[g] - at;
#pragma unroll
                for (int i = 0; i < (int)VER_N; ++i) e[i] = d == (uint32_t)i ? 0.0 : e[i];
            }
        };
        for (;;) {
            if (plain) {
                for (uint32_t c = tid; c < a.nc; c += VER_T) {
                    const VerPart q = a.tp[row * a.nc + c];
                    sums[c] = q.z * weight(q.m, f.tm, it);
                }
                __syncthreads();
                // chunks that lose tokens are summed again: what is left may be much less than what goes
                for (uint32_t g = 0; g < cut; ++g) {
                    if (gone[g] >= p.vocab) continue;
                    const uint32_t c = gone[g] / VER_CH;
                    bool seen = false;
                    for (uint32_t h = 0; h < g; ++h) seen = seen || (gone[h] < p.vocab && gone[h] / VER_CH == c);
                    if (seen) continue;
                    chunk(c);
                    double v = 0;
#pragma unroll
                    for (int i = 0; i < (int)VER_N; ++i) v += e[i];
                    v = wg_sum(v, sm);
                    if (tid == 0) sums[c] = v;
                }
                __syncthreads();
            }
            if (tid < 64) {                                           // the chunk, by one wave
                double all = 0;
                for (uint32_t c = tid; c < a.nc; c += 64) all += sums[c];
                all = wave_sum(all);
                const double want = p.u_next[s] * all;
                double before = 0;
                uint32_t pick = NO_ROW, most = NO_ROW;
                double most_before = 0;
                for (uint32_t c0 = 0; c0 < a.nc && pick == NO_ROW; c0 += 64) {
                    const uint32_t c = c0 + tid;
                    const double v = c < a.nc ? sums[c] : 0.0;
                    double in = v;
#pragma unroll
                    for (int d = 1; d < 64; d <<= 1) {
                        const double o = __shfl_up(in, d);
                        if (tid >= (uint32_t)d) in += o;
                    }
                    const uint64_t hit = __ballot(before + in > want && v > 0), some = __ballot(v > 0);
                    const int l = hit ? __builtin_ctzll(hit) : some ? 63 - __builtin_clzll(some) : 0;
                    const double at = before + __shfl(in - v, l);
                    if (hit) {
                        pick = c0 + l;
                        before = at;
                    } else {
                        if (some) { most = c0 + l; most_before = at; }
                        before += __shfl(in, 63);
                    }
                }
                if (pick == NO_ROW) { pick = most; before = most_before; }    // (rounding: the last one with weight)
                if (tid == 0) {
                    sm_pick = pick;
                    sm[0] = want - before;
                }
            }
            __syncthreads();
            if (sm_pick != NO_ROW || !cut) break;
            cut = 0;                                                  // the tokens taken out were all there is: p itself
            __syncthreads();
        }
        const uint32_t c = sm_pick;
        const double want = sm[0];
        __syncthreads();
        if (c != NO_ROW) {
            chunk(c);
            double v = 0;
#pragma unroll
            for (int i = 0; i < (int)VER_N; ++i) v += e[i];
            double in = v;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const double o = __shfl_up(in, d);
                if ((tid & 63) >= (uint32_t)d) in += o;
            }
            if ((tid & 63) == 63) sm[tid >> 6] = in;
            if (tid == 0) sm_pick = NO_ROW;
            __syncthreads();
            for (uint32_t i = 0; i < tid >> 6; ++i) in += sm[i];
            // the first token whose sum passes the number; none (rounding): the last one with weight
            uint32_t hit = NO_ROW, last = 0;
            double at = in - v;
#pragma unroll
            for (int i = 0; i < (int)VER_N; ++i) {
                at += e[i];
                if (e[i] > 0) {
                    last = c * VER_CH + tid * VER_N + i + 1;
                    if (hit == NO_ROW && at > want) hit = last - 1;
                }
            }
            if (hit != NO_ROW) atomicMin(&sm_pick, hit);
            if (tid == 0) sm_last = 0;
            __syncthreads();
            if (last) atomicMax(&sm_last, last);
            __syncthreads();
            next = sm_pick != NO_ROW ? sm_pick : sm_last - 1;
        }
    }
    // ---- outputs: the path from its end (a thread), the other places
    for (uint32_t j = w.len + tid; j < p.path_stride; j += VER_T) {
        p.path[out + j] = FLH_KV_NONE;
        if (p.logp) p.logp[out + j] = 0.f;
    }
    if (tid == 0) {
        uint32_t cur = end;
        double lp = 0;
        if (!greedy && next != FLH_KV_NONE) lp = ((double)logit((float)xr[next]) - (double)tr.m) * it - log(tr.z);
        for (uint32_t j = w.len; j-- > 0;) {
            p.path[out + j] = cur;
            if (p.logp) p.logp[out + j] = (float)lp;
            lp = greedy ? 0.0 : log(w.pc[cur]);
            cur = w.up[cur];
        }
        p.n_path[s] = w.len;
        p.next[s] = next;
        if (p.len) p.len[s] = p.kv_len[s] - (p.q_start[s + 1] - p.q_start[s]) + w.len;
    }
}

// ----------------------------------------------------------------- launches --
static void verify_plan(const flh_verify_p & p, VerArgs & a, size_t & bytes) {
    a = VerArgs{};
    a.p = p;
    a.nc = (p.vocab + VER_CH - 1) / VER_CH;
    a.share = p.draft ? a.nc : 1;
    a.rounds = p.draft && p.parent && p.max_child > 1 ? p.max_child - 1 : 0;
    const uint64_t parts = (uint64_t)p.n_tok * a.nc;
    uint8_t * at = (uint8_t *)p.ws;
    size_t n = 0;
    auto take = [&](uint64_t b) {
        uint8_t * r = at + n;
        n += (b + 15) & ~(uint64_t)15;
        return r;
    };
    a.tp = (VerPart *)take(parts * sizeof(VerPart));
    if (p.draft) {
        a.dp = (VerPart *)take(parts * sizeof(VerPart));
        a.rest = (double *)take(a.rounds * parts * 8);
        a.left = (double *)take((uint64_t)p.n_seq * a.nc * 8);
        a.done = (uint32_t *)take((uint64_t)p.n_seq * 4);
    }
    bytes = n;
}
size_t verify_ws_bytes(const flh_verify_p & p) {
    VerArgs a;
    size_t n;
    verify_plan(p, a, n);
    return n;
}
template <typename T> static int verify_go(const VerArgs & a, hipStream_t s) {
    const uint32_t rows = a.p.n_tok * a.nc;
    if (rows) {
        hipLaunchKernelGGL(k_verify_sums<T>, dim3(rows, a.p.draft ? 2 : 1), dim3(VER_T), 0, s, a);
        if (int rc = hip_check(hipGetLastError(), "k_verify_sums launch")) return rc;
        for (uint32_t i = 1; i <= a.rounds; ++i) {
            hipLaunchKernelGGL(k_verify_rest<T>, dim3(rows), dim3(VER_T), 0, s, a, i);
            if (int rc = hip_check(hipGetLastError(), "k_verify_rest launch")) return rc;
        }
    }
    hipLaunchKernelGGL(k_verify_next<T>, dim3(a.p.n_seq * a.share), dim3(VER_T), 0, s, a);
    return hip_check(hipGetLastError(), "k_verify_next launch");
}
int launch_verify(const flh_verify_p & p, hipStream_t s) {
    VerArgs a;
    size_t n;
    verify_plan(p, a, n);
    if (p.dtype == FLH_DT_F32) return verify_go<float>(a, s);
    return p.dtype == FLH_DT_F16 ? verify_go<_Float16>(a, s) : verify_go<__bf16>(a, s);
}

}  // namespace flh
