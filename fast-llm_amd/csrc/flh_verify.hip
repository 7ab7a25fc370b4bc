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
// Launches: sums of every row's chunks; n_i (only with several children a row); the walk and the
// draw.  A random number may lie next to the border of two of 10^5 tokens, so weights, sums and
// borders are in 64 bits: with the exponential below an element costs 17 instructions of a
// SIMD, about as much time as its bytes in fp32.
#include "flh_common.h"
#include "flh_internal.h"
#include "flh_status.h"
#include <float.h>
#include <type_traits>

namespace flh {

constexpr int VER_N = 16;
constexpr uint32_t VER_T = 256, VER_CH = VER_T * VER_N;   // threads, elements a thread, of a chunk
constexpr uint32_t VER_ROWS = 256;                                    // of a request that are looked at
constexpr uint32_t NO_ROW = 0xFFFFFFFFu;

// A chunk's largest logit, where it first is (greedy requests), and the sum of
// exp((x - m) inv_temp).
struct VerPart {
    double z;
    float m;
    uint32_t at;
};
// A row's request's inv_temp, and the row's children (0 for a row of none)
struct VerMeta {
    float it;
    uint32_t kids;
};
struct VerArgs {
    flh_verify_p p;
    VerPart * tp, * dp;                 // [n_tok][nc]
    VerMeta * meta;                     // [n_tok] (with a draft)
    double * rest;                      // [max_child - 1][n_tok][nc]: n_1 ..
    double * left;                      // [n_seq][nc]
    uint32_t * done;                    // [n_seq]
    uint32_t nc, rounds, share;         // chunks of a row; launches of k_verify_rest; workgroups of a request's draw
};

// The weights exp((x - m) inv_temp) = 2^((x - m) c) of a row's logits, m the largest of them (0 in its place where
// it is -infinity).  2^y = 2^k 2^f: adding 1.5 * 2^52 leaves the nearest whole number in the low bits, so k needs no
// conversion and goes into the exponent by an integer addition; 2^f, |f| <= 1/2, by the polynomial that takes its
// values at the ten Chebyshev points of the interval (off by 1.9e-14 of the value at most).  Below 2^-1000: 0.
struct VerExp {
    double m, c;
    __device__ __forceinline__ VerExp() {}
    __device__ __forceinline__ VerExp(float top, double it) : m(top == -INFINITY ? 0.0 : (double)top), c(it * 1.4426950408889634074) {}
    // 2^f times 2^(the whole number in t's low bits), several at once: an instruction waits for the one before it
    // about four times as long as it takes
    template <int N> __device__ __forceinline__ static void pow2(const double (&f)[N], const double (&t)[N], double (&e)[N]) {
        constexpr double a[10] = {0x1.000000000003dp+0, 0x1.62e42fefa39f7p-1, 0x1.ebfbdff8149f2p-3, 0x1.c6b08d7044119p-5,
                                  0x1.3b2ab72b175eep-7, 0x1.5d87fe908f88ap-10, 0x1.43088e257f341p-13, 0x1.ffcb76789860fp-17,
                                  0x1.63ef969a64d3cp-20, 0x1.b6571de2f2351p-24};
#pragma unroll
        for (int i = 0; i < N; ++i) e[i] = fma(a[9], f[i], a[8]);
#pragma unroll
        for (int j = 7; j >= 0; --j) {
#pragma unroll
            for (int i = 0; i < N; ++i) e[i] = fma(e[i], f[i], a[j]);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) e[i] = __hiloint2double(__double2hiint(e[i]) + (__double2loint(t[i]) << 20), __double2loint(e[i]));
    }
    static constexpr double MAGIC = 6755399441055744.0;
    template <int N> __device__ __forceinline__ void of(const float (&x)[N], double (&e)[N]) const {
        double y[N], t[N], f[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            y[i] = fmax(((double)x[i] - m) * c, -1000.0);             // (-infinity times an inv_temp of 0: here, too)
            t[i] = y[i] + MAGIC;
            f[i] = y[i] - (t[i] - MAGIC);
        }
        pow2<N>(f, t, e);
#pragma unroll
        for (int i = 0; i < N; ++i) e[i] = y[i] <= -1000.0 ? 0.0 : e[i];
    }
    __device__ __forceinline__ double of(float x) const {
        const float y[1] = {x};
        double e[1];
        of<1>(y, e);
        return e[0];
    }
    // The same with fewer instructions, for a sum that has a 1 in it: of logits that are at least `low`, whose weight, about
    // 2^-600, makes no difference.  (false: m is so large, or inv_temp so small, that no float is that far below it.)
    __device__ __forceinline__ bool lowest(float top, float & low) const {
        low = top - 600.f / (float)c;
        const double y = ((double)low - (double)top) * c;
        return y >= -1000.0 && y <= -100.0;
    }
    template <int N> __device__ __forceinline__ void rough(const float (&x)[N], double (&e)[N]) const {
        double t[N], f[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const double d = (double)x[i] - m;
            t[i] = fma(d, c, MAGIC);
            f[i] = fma(d, c, MAGIC - t[i]);
        }
        pow2<N>(f, t, e);
    }
};
// A logit as it is in memory.  One that is no number is a quiet one behind this: of a signalling one the instructions below
// make a quiet one first and then the other operand, which would be the largest number.  The conversion from f16
// quiets by itself; the compiler would leave a multiplication by 1 out.
template <typename T> __device__ __forceinline__ float number(T x) {
    if constexpr (std::is_same_v<T, _Float16>) return (float)x;
    float y;
    asm("v_max_f32 %0, %1, %1" : "=v"(y) : "v"((float)x));
    return y;
}
// What is no number counts as -infinity, infinity as the largest number: the median of three, which is their
// smallest where one is no number.  (In asm: the compiler takes the median with -infinity for a minimum of two, which
// makes the largest number of what is none.)
__device__ __forceinline__ float logit(float x, float low = -INFINITY) {
    float y;
    asm("v_med3_f32 %0, %1, %2, %3" : "=v"(y) : "v"(x), "v"(low), "s"(FLT_MAX));
    return y;
}
// the largest of three that is a number (in asm: the compiler would look for signalling ones first), or, MUST, no number where one is none
template <bool MUST = false> __device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    if constexpr (MUST) asm("v_maximum3_f32 %0, %1, %2, %3" : "=v"(y) : "v"(a), "v"(b), "v"(c));
    else asm("v_max3_f32 %0, %1, %2, %3" : "=v"(y) : "v"(a), "v"(b), "v"(c));
    return y;
}
// Sums, maxima and minima over groups of G lanes, the same in each of them (all lanes of the wave are on), without
// LDS: a permute through it takes longer than the addition.
__device__ __forceinline__ double xor_lane64(double v, int o, uint32_t lane) {
    const float lo = xor_lane(__int_as_float(__double2loint(v)), o, lane), hi = xor_lane(__int_as_float(__double2hiint(v)), o, lane);
    return __hiloint2double(__float_as_int(hi), __float_as_int(lo));
}
template <int G = 64> __device__ __forceinline__ double group_sum(double v) {
    const uint32_t lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < G; d <<= 1) v += xor_lane64(v, d, lane);
    return v;
}
template <int G = 64> __device__ __forceinline__ float group_max(float v) {
    const uint32_t lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < G; d <<= 1) v = fmaxf(v, xor_lane(v, d, lane));
    return v;
}
template <int G = 64> __device__ __forceinline__ uint32_t group_min(uint32_t v) {
    const uint32_t lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < G; d <<= 1) v = min(v, __float_as_uint(xor_lane(__uint_as_float(v), d, lane)));
    return v;
}
// Inclusive sums over the wave's lanes: within rows of 16, then the rows before.
template <int N> __device__ __forceinline__ double lane_before(double v) {     // 0 in a row's first N lanes
    return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(v), 0x110 + N, 0xF, 0xF, false),
                            __builtin_amdgcn_update_dpp(0, __double2loint(v), 0x110 + N, 0xF, 0xF, false));
}
__device__ __forceinline__ double lane_at(double v, int l) {
    return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), l), __builtin_amdgcn_readlane(__double2loint(v), l));
}
__device__ __forceinline__ double wave_scan(double v) {
    const uint32_t lane = threadIdx.x & 63;
    v += lane_before<1>(v);
    v += lane_before<2>(v);
    v += lane_before<4>(v);
    v += lane_before<8>(v);
    const double a = lane_at(v, 15), b = a + lane_at(v, 31), c = b + lane_at(v, 47);
    return v + (lane >= 48 ? c : lane >= 32 ? b : lane >= 16 ? a : 0.0);
}

// A thread's elements of a chunk that W waves share, as they are in memory, in pieces of 16 bytes: a wave's lie
// together, lane by lane (IN_ORDER: a thread's own).  A piece that reaches behind the row's end is read from in front of
// it, so that no lane takes a branch, at whose end the loads would wait for one another; its elements that are
// another piece's count as -infinity.
template <typename T, bool IN_ORDER, int W = 4> struct Chunk {
    static constexpr int N = 16 / sizeof(T), E = VER_CH / 64 / W;
    struct alignas(sizeof(T)) V { T v[N]; };
    V t[E / N];
    __device__ __forceinline__ static uint32_t at(uint32_t c, int j) {
        return IN_ORDER ? c * VER_CH + threadIdx.x * E + j * N
                        : c * VER_CH + (threadIdx.x >> 6) * 64 * E + (j * 64 + (threadIdx.x & 63)) * N;
    }
    __device__ __forceinline__ void load(const T * row, uint32_t c, uint32_t v) {
        if (v < N) {                                                  // (uniform: hardly a vocabulary)
#pragma unroll
            for (int i = 0; i < N; ++i) t[0].v[i] = row[min((uint32_t)i, v - 1)];
            return;
        }
#pragma unroll
        for (int j = 0; j < E / N; ++j) __builtin_memcpy(&t[j], row + min(at(c, j), v - N), sizeof t[j]);
    }
    // the logits (RAW: as they are), and which token element e is
    template <bool RAW = false> __device__ __forceinline__ void get(uint32_t c, uint32_t v, float (&x)[E]) const {
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = RAW ? (float)t[e / N].v[e % N] : logit(number(t[e / N].v[e % N]));
        if ((c + 1) * VER_CH <= v) return;                            // (uniform)
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const uint32_t k = token(c, v, e);
            x[e] = k >= at(c, e / N) && k < v ? x[e] : -INFINITY;
        }
    }
    __device__ __forceinline__ static uint32_t token(uint32_t c, uint32_t v, int e) {
        return min(at(c, e / N), v < N ? 0u : v - N) + e % N;
    }
};
// Sum over the workgroup, the same in every thread (sm: 4 values; waves are added in order)
__device__ __forceinline__ double wg_sum(double v, double * sm) {
    v = group_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = v;
    __syncthreads();
    return sm[0] + sm[1] + sm[2] + sm[3];
}

__device__ __forceinline__ double inv_temp_of(const flh_verify_p & p, uint32_t s) {
    const float it = p.inv_temp ? p.inv_temp[s] : 1.f;
    return it >= 0.f ? (double)it : 0.0;                              // (infinity: greedy)
}
// rows of a request that are looked at, from its first and the next one's
__device__ __forceinline__ uint32_t rows_of(const flh_verify_p & p, uint32_t & r0, uint32_t end) {
    r0 = min(r0, p.n_tok);
    end = min(end, p.n_tok);
    return end > r0 ? min(end - r0, VER_ROWS) : 0u;
}
// A row's request: its inv_temp, its rows and where they begin
struct VerReq {
    double it;
    uint32_t r0, n;
};
// The request of a row (false: of none), the last one that begins at or before it, by a wave that looks at 64 of
// them at once: one round of loads for up to 63 requests, two or three for 4000.
__device__ __forceinline__ bool request_of(const flh_verify_p & p, uint32_t row, VerReq & r) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t lo = 0, n = p.n_seq + 1, k;
    while (n > 64) {
        const uint32_t step = (n + 63) / 64, i = lane * step;
        const uint32_t first = p.q_start[lo + (i < n ? i : 0)];
        k = (uint32_t)__popcll(__ballot(i < n && first <= row));
        if (k == 0) return false;
        lo += (k - 1) * step;
        n = min(step + 1, n - (k - 1) * step);                        // (and where the next one begins)
    }
    const uint32_t at = lo + min(lane, n - 1), first = p.q_start[at];
    const float mine = p.inv_temp ? p.inv_temp[min(at, p.n_seq - 1)] : 1.f;
    k = (uint32_t)__popcll(__ballot(lane < n && first <= row));
    if (k == 0 || lo + k > p.n_seq) return false;
    // (where the others begin out of order, k may be n)
    const float it = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(mine), k - 1));
    r.it = it >= 0.f ? (double)it : 0.0;
    r.r0 = __builtin_amdgcn_readlane(first, k - 1);
    r.n = rows_of(p, r.r0, k < n ? (uint32_t)__builtin_amdgcn_readlane(first, k & 63) : p.q_start[lo + k]);
    return true;
}
// the row that row i of a request hangs on (NO_ROW: none)
__device__ __forceinline__ uint32_t parent_of(const flh_verify_p & p, uint32_t r0, uint32_t i) {
    const uint32_t x = p.parent ? (uint32_t)p.parent[r0 + i] : i - 1;
    return x < i ? x : NO_ROW;
}
// children of row i of a request of n rows (at most max_child), by a wave
__device__ __forceinline__ uint32_t children(const flh_verify_p & p, uint32_t r0, uint32_t n, uint32_t i) {
    if (!p.parent) return i + 1 < n;
    uint32_t k = 0;
    for (uint32_t j0 = i + 1; j0 < n; j0 += 64) {
        const uint32_t j = j0 + (threadIdx.x & 63);
        k += (uint32_t)__popcll(__ballot(j < n && parent_of(p, r0, min(j, n - 1)) == i));
    }
    return min(k, p.max_child);
}

// ------------------------------------------------------------- the rows' sums --
// Workgroup (row, side, chunk) of the target or of the draft (rows with children), two waves.  Instructions bound it:
// 17 an element, 15 of them in 64 bits, and 110 a wave for whose row it is and for putting the sums together, so a thread has 32 elements (with 16
// they take 28 us for 32 requests of 2 to 6 rows of 128256 with a draft, so 25).  Longer shares, the next chunk's logits on their way
// meanwhile, leave the last workgroups alone for longer than they save.  The target's logits are asked for before it is known
// whose they are, but only of rows that some request may have: of a captured step with room for four times as many rows the
// others would be most of the bytes (32 chains 69 us, 48 so; without spare rows 42.5 and 43).
constexpr int SUM_W = 2;
template <typename T> __global__ __launch_bounds__(64 * SUM_W) void k_verify_sums(VerArgs a) {
    typedef Chunk<T, false, SUM_W> C;
    __shared__ float sm_m;
    __shared__ double sm_z;
    __shared__ uint32_t sm_at;
    const flh_verify_p & p = a.p;
    const uint32_t lane = threadIdx.x & 63, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t side = blockIdx.x / a.nc, c = blockIdx.x - side * a.nc, row = p.draft ? side >> 1 : side;
    const bool draft = p.draft && (side & 1);
    if (blockIdx.x == 0 && p.draft)
        for (uint32_t i = threadIdx.x; i < p.n_seq; i += 64 * SUM_W) a.done[i] = 0;
    C chunk;
    if (!draft) {
        if (row >= p.q_start[p.n_seq]) return;                        // (uniform)
        chunk.load((const T *)p.target + row * p.t_row, c, p.vocab);
    }
    VerReq q;
    const bool some = request_of(p, row, q);
    if (draft) {
        const uint32_t kids = some && !isinf(q.it) && row - q.r0 < q.n ? children(p, q.r0, q.n, row - q.r0) : 0;
        if (c == 0 && threadIdx.x == 0) a.meta[row] = VerMeta{(float)q.it, kids};
        if (kids == 0) return;
        chunk.load((const T *)p.draft + row * p.d_row, c, p.vocab);
    }
    if (!some) return;
    const bool greedy = isinf(q.it);
    float x[C::E];
    chunk.template get<true>(c, p.vocab, x);
    VerPart o{0, -INFINITY, NO_ROW};
#pragma unroll
    for (int i = 0; i < C::E; i += 2) o.m = max3<true>(o.m, x[i], x[i + 1]);
    if (__ballot(isnan(o.m))) {                                       // (hardly ever: 43 us for 32 chains instead of 44 with `number` for all)
        o.m = -INFINITY;
#pragma unroll
        for (int i = 0; i < C::E; ++i) x[i] = number(x[i]);
#pragma unroll
        for (int i = 0; i < C::E; i += 2) o.m = max3(o.m, x[i], x[i + 1]);
    }
    o.m = group_max(fminf(o.m, FLT_MAX));
    if (greedy) {
#pragma unroll
        for (int i = C::E - 1; i >= 0; --i) o.at = logit(x[i]) == o.m && o.m > -INFINITY ? min(o.at, chunk.token(c, p.vocab, i)) : o.at;
        o.at = group_min(o.at);
    } else {
        const VerExp e(o.m, q.it);
        double z[4] = {0, 0, 0, 0}, g[4];
        float low;
        if (e.lowest(o.m, low)) {
#pragma unroll
            for (int i = 0; i < C::E; i += 4) {
                const float y[4] = {logit(x[i], low), logit(x[i + 1], low), logit(x[i + 2], low), logit(x[i + 3], low)};
                e.template rough<4>(y, g);
#pragma unroll
                for (int j = 0; j < 4; ++j) z[j] += g[j];
            }
        } else if (o.m > -INFINITY) {
            for (int i = 0; i < C::E; ++i) z[0] += e.of(logit(x[i]));
        }
        o.z = group_sum((z[0] + z[1]) + (z[2] + z[3]));
    }
    if (wave == 1 && lane == 0) {
        sm_m = o.m;
        sm_z = o.z;
        sm_at = o.at;
    }
    __syncthreads();
    if (threadIdx.x) return;
    const float m = fmaxf(o.m, sm_m);
    const VerExp e(m, greedy ? 1.0 : q.it);
    const float y[2] = {o.m, sm_m};
    double g[2];
    e.of(y, g);
    (draft ? a.dp : a.tp)[(uint64_t)row * a.nc + c] =
        VerPart{o.z * g[0] + sm_z * g[1], m, min(o.m == m ? o.at : NO_ROW, sm_m == m ? sm_at : NO_ROW)};
}

// A row's largest logit and sum from its chunks', by the lanes of a group of G in step; and
// where the largest first is
struct VerRow {
    float m;
    double z;
    uint32_t at;
};
template <int G> __device__ __forceinline__ VerRow merge_row(const VerPart * part, uint32_t nc, double it) {
    constexpr uint32_t N = G < 8 ? 8 : 2;                             // parts a lane takes at once
    const uint32_t l = threadIdx.x % G;
    VerRow r{-INFINITY, 0.0, NO_ROW};
    for (uint32_t c0 = 0; c0 < nc; c0 += N * G) {
        VerPart q[N];
        float m = r.m;
#pragma unroll
        for (uint32_t j = 0; j < N; ++j) q[j] = part[min(c0 + l + j * G, nc - 1)];
#pragma unroll
        for (uint32_t j = 0; j < N; ++j) m = fmaxf(m, q[j].m);
        m = group_max<G>(m);
        const VerExp e(m, it);
        r.at = r.m == m ? r.at : NO_ROW;
        r.z *= e.of(r.m);
#pragma unroll
        for (uint32_t j = 0; j < N; ++j) {
            r.at = q[j].m == m ? min(r.at, q[j].at) : r.at;
            const double z = q[j].z * e.of(q[j].m);
            r.z += c0 + l + j * G < nc ? z : 0.0;
        }
        r.m = m;
    }
    r.z = group_sum<G>(r.z);
    r.at = group_min<G>(r.at);
    return r;
}
// n_j of a row (j >= 1), and t_i = 1 + n_1 + .. + n_(i-1) (i >= 1), by the lanes of a group of G in step
template <int G> __device__ __forceinline__ double rest_of(const VerArgs & a, uint32_t row, uint32_t j) {
    constexpr uint32_t N = G < 8 ? 8 : 2;
    const double * r = a.rest + ((uint64_t)(j - 1) * a.p.n_tok + row) * a.nc;
    double n = 0;
    for (uint32_t c0 = threadIdx.x % G; c0 < a.nc; c0 += N * G) {
        double v[N];
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) v[i] = r[min(c0 + i * G, a.nc - 1)];
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) n += c0 + i * G < a.nc ? v[i] : 0.0;
    }
    return group_sum<G>(n);
}
template <int G> __device__ __forceinline__ double taken_of(const VerArgs & a, uint32_t row, uint32_t i) {
    double t = 1.0;
    for (uint32_t j = 1; j < i; ++j) t += rest_of<G>(a, row, j);
    return t;
}
__device__ __forceinline__ double total(const double (&w)[VER_N]) {
    double v[4] = {w[0], w[1], w[2], w[3]};
#pragma unroll
    for (int i = 4; i < VER_N; ++i) v[i & 3] += w[i];
    return (v[0] + v[1]) + (v[2] + v[3]);
}
// What is left of p: max(p - t q, 0) of tokens' two logits.  (Both products are rounded: a draft that is
// the target leaves nothing, not the rounding of one of them.)
struct VerLeft {
    VerExp p, q;
    double fp, fq;
    __device__ __forceinline__ void of(const float (&x)[VER_N], const float (&y)[VER_N], double (&w)[VER_N]) const {
#pragma unroll
        for (int i = 0; i < VER_N; i += 4) {
            const float x4[4] = {x[i], x[i + 1], x[i + 2], x[i + 3]}, y4[4] = {y[i], y[i + 1], y[i + 2], y[i + 3]};
            double g[4], h[4];
            p.of<4>(x4, g);
            q.of<4>(y4, h);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[i + j] = fmax(g[j] * fp - h[j] * fq, 0.0);
        }
    }
};
__device__ __forceinline__ VerLeft left_of(const VerRow & t, const VerRow & d, double taken, double it) {
    return VerLeft{VerExp(t.m, it), VerExp(d.m, it), t.z > 0 ? 1.0 / t.z : 0.0, d.z > 0 ? taken / d.z : 0.0};
}

// n_i, i = `round`, of the rows with more than i children: workgroup (row, chunk).  Its waves put the row's sums
// together, one each, while the logits are on their way.  16 requests of 7 to 21 rows, 50257 tokens in bf16: 14 us, of
// which the instructions of two exponentials an element are about 4 and three rounds of loads the rest.
template <typename T> __global__ __launch_bounds__(VER_T) void k_verify_rest(VerArgs a, uint32_t round) {
    __shared__ double sm[4], sm_z[2], sm_t;
    __shared__ float sm_m[2];
    const flh_verify_p & p = a.p;
    const uint32_t row = blockIdx.x / a.nc, c = blockIdx.x - row * a.nc, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const VerMeta q = a.meta[row];
    if (q.kids <= round) return;
    const double it = q.it;
    Chunk<T, false> xc, yc;
    xc.load((const T *)p.target + row * p.t_row, c, p.vocab);
    yc.load((const T *)p.draft + row * p.d_row, c, p.vocab);
    if (wave < 2) {
        const VerRow r = merge_row<64>((wave ? a.dp : a.tp) + (uint64_t)row * a.nc, a.nc, it);
        sm_m[wave] = r.m;
        sm_z[wave] = r.z;
    } else if (wave == 2) sm_t = taken_of<64>(a, row, round);
    __syncthreads();
    const VerLeft f = left_of(VerRow{sm_m[0], sm_z[0], 0}, VerRow{sm_m[1], sm_z[1], 0}, sm_t, it);
    float x[VER_N], y[VER_N];
    xc.get(c, p.vocab, x);
    yc.get(c, p.vocab, y);
    double w[VER_N];
    f.of(x, y, w);
    const double sum = wg_sum(total(w), sm);
    if (threadIdx.x == 0) a.rest[((uint64_t)(round - 1) * p.n_tok + row) * a.nc + c] = sum;
}

// -------------------------------------------------------- the walk and the draw --
// A thread a row: its parent, its token and what its test needs are asked for at once, before the
// rows' sums are put together (16 lanes a row), so the walk is three rounds of loads long.  With a draft every
// workgroup of a request (one a chunk) walks by itself, then sums what is left of its chunk of the row at the path's end; the last
// one to finish draws: 17 to 19 us for 32 requests of 128256 tokens, 8 to 10 for one without a draft.  Rounds of loads bound it.
struct VerWalk {
    double tz[VER_ROWS], dz[VER_ROWS], pc[VER_ROWS];                  // sums of rows; p of rows' tokens
    double t[VER_ROWS], n[VER_ROWS];                                  // what rows' tests are against
    float tm[VER_ROWS], dm[VER_ROWS];
    uint32_t at[VER_ROWS], up[VER_ROWS], best[VER_ROWS], tok[VER_ROWS];   // where rows' largest are; parents; first child that stands
    uint8_t rank[VER_ROWS], path[VER_ROWS];                           // among its siblings (255: behind max_child, none)
    uint32_t len, k;                                                  // the path's rows; whether the last one's children count
};

template <typename T> __global__ __launch_bounds__(VER_T) void k_verify_next(VerArgs a) {
    __shared__ VerWalk w;
    __shared__ double sm[4], sums[1024], gone_e[64];
    __shared__ uint32_t sm_last, sm_pick, gone[64], again[64], n_again;
    __shared__ float sm_x;
    const flh_verify_p & p = a.p;
    const uint32_t s = blockIdx.x / a.share, part = blockIdx.x % a.share, tid = threadIdx.x;
    const double it = inv_temp_of(p, s);
    const bool greedy = isinf(it);
    const double wt = greedy ? 1.0 : it;                              // (a finite one for sums that nobody reads)
    uint32_t r0 = p.q_start[s];
    const uint32_t rows = p.q_start[s + 1] - r0, n = rows_of(p, r0, r0 + rows);
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
            if (p.len) p.len[s] = p.kv_len[s] - rows;                 // (rows that n_tok cuts off have no keys)
        }
        return;
    }
    const float u_next = p.u_next[s];
    // ---- the rows: what hangs on what, and their logits at their parents
    // (loads of a place that is there and selects: a branch that some lanes take would wait for its loads)
    const uint32_t mine = min(tid, n - 1);
    const uint32_t hangs = p.parent ? (uint32_t)p.parent[r0 + mine] : tid - 1, tok = p.token[r0 + mine];
    const float u = p.u_accept[r0 + mine];
    const uint32_t up = tid < n && hangs < tid ? hangs : NO_ROW;
    const bool drafted = up != NO_ROW && tok < p.vocab;
    const T * xa = (const T *)p.target + (uint64_t)r0 * p.t_row;
    const T * ya = drafted && p.draft && !greedy ? (const T *)p.draft + (r0 + up) * p.d_row + tok : xa;
    xa += drafted ? up * p.t_row + tok : 0;
    const T xt = *xa, yt = *ya;
    w.up[tid] = up;
    w.best[tid] = NO_ROW;
    w.tok[tid] = tok;
    // (a draft's row without children: anything, and not used)
    const bool drafts = p.draft && !greedy;
    const uint32_t merges = drafts ? 2 * n : n;
    auto merge = [&](auto lanes) {                                    // a row's parts by so many lanes
        constexpr uint32_t G = decltype(lanes)::value;
        for (uint32_t i0 = 0; i0 < merges; i0 += VER_T / G) {
            if (i0 + (tid & ~63u) / G >= merges) break;               // (no row for this wave)
            const uint32_t x = i0 + tid / G;
            const bool d = x >= n && drafts;
            const uint32_t i = min(d ? x - n : x, n - 1);
            const VerRow r = merge_row<G>((d ? a.dp : a.tp) + (uint64_t)(r0 + i) * a.nc, a.nc, wt);
            (d ? w.dm : w.tm)[i] = r.m;
            (d ? w.dz : w.tz)[i] = r.z;
            if (!d) w.at[i] = r.at;
        }
    };
    if (merges <= VER_T / 16) merge(std::integral_constant<int, 16>());
    else merge(std::integral_constant<int, 4>());
    __syncthreads();
    uint32_t rank = 0;
    if (p.parent && up != NO_ROW)
        for (uint32_t j = up + 1; j < tid; ++j) rank += w.up[j] == up;
    const bool tested = up != NO_ROW && rank < p.max_child;
    w.rank[tid] = tested ? (uint8_t)rank : 255;
    // ---- p of the rows' tokens
    const float xl = logit(number(xt)), yl = logit(number(yt));
    double e = 0, pc = 0;
    if (drafted) {
        e = greedy ? 0.0 : VerExp(w.tm[up], it).of(xl);
        pc = greedy ? (w.at[up] == tok ? 1.0 : 0.0) : w.tz[up] > 0 ? e / w.tz[up] : 0.0;
    }
    w.pc[tid] = pc;
    if (a.rounds) {                                                   // (rows of one child each: t is 0, n is 1)
        __syncthreads();
        if (!greedy)
            for (uint32_t i0 = 0; i0 < n; i0 += VER_T / 4) {
                const uint32_t i = min(i0 + tid / 4, n - 1), k = w.rank[i] == 255 ? 0 : w.rank[i];
                double t = 0, m = 1;
                for (uint32_t j = 1; __ballot(j <= k); ++j) {         // (the groups of a wave together)
                    const double r = rest_of<4>(a, r0 + (j <= k ? w.up[i] : 0), j);
                    t = j <= k ? t + m : t;
                    m = j <= k ? r : m;
                }
                w.t[i] = t;
                w.n[i] = m;
            }
    }
    __syncthreads();
    // ---- which rows stand against their parent's distribution
    if (tested) {
        bool ok;
        if (greedy) ok = pc > 0;
        else if (p.draft) {
            double qc = 0;
            if (drafted && w.dz[up] > 0) qc = VerExp(w.dm[up], it).of(yl) / w.dz[up];
            const double t = rank ? w.t[tid] : 0.0, m = rank ? w.n[tid] : 1.0;
            ok = u * qc * m < fmax(pc - t * qc, 0.0);
        } else {
            double took = 0;
            bool twice = false;
            if (rank)
                for (uint32_t j = up + 1; j < tid; ++j) {
                    if (w.up[j] != up) continue;
                    bool before = false;
                    for (uint32_t l = up + 1; l < j; ++l) before = before || (w.up[l] == up && w.tok[l] == w.tok[j]);
                    twice = twice || w.tok[j] == tok;
                    if (!before) took += w.pc[j];
                }
            ok = !twice && u * (1.0 - took) < pc;
        }
        if (ok) atomicMin(&w.best[up], tid);
    }
    __syncthreads();
    // ---- the path: from row 0 on, the first child that stands
    if (tid == 0) {
        uint32_t cur = 0, len = 1;
        w.path[0] = 0;
        while (len < p.path_stride && w.best[cur] != NO_ROW) {
            cur = w.best[cur];
            w.path[len++] = (uint8_t)cur;
        }
        w.len = len;
        // (A path cut off ends as at a row without children, whether one of them would have stood or not: drawn from what
        // is left where none would, the token would not be distributed as p.)
        w.k = len < p.path_stride;
        n_again = 0;
    }
    __syncthreads();
    const uint32_t len = w.len, end = w.path[len - 1];
    const uint64_t row = r0 + end;
    // its children, which do not stand
    const bool lost = w.k && up == end && tested;
    const uint32_t k = greedy ? 0 : (uint32_t)__syncthreads_count(lost);
    const bool both = p.draft && k;                                   // what is left of p takes a pass over the row
    if (part && !both) return;
    if (!p.draft && lost) {                                           // their tokens (each once) and weights, by rank
        bool twice = false;
        for (uint32_t j = end + 1; j < tid; ++j) twice = twice || (w.up[j] == end && w.tok[j] == tok);
        gone[rank] = drafted && !twice ? tok : NO_ROW;
        gone_e[rank] = e;
    }
    const VerRow tr{w.tm[end], w.tz[end], w.at[end]}, dr{w.dm[end], w.dz[end], 0};
    const T * xr = (const T *)p.target + row * p.t_row;
    const T * yr = both ? (const T *)p.draft + row * p.d_row : nullptr;
    bool plain = !both;
    VerLeft f;
    f.p = VerExp(tr.m, wt);
    if (both) {
        float x[VER_N], y[VER_N];
        Chunk<T, false> xc, yc;
        xc.load(xr, part, p.vocab);
        yc.load(yr, part, p.vocab);
        xc.get(part, p.vocab, x);
        yc.get(part, p.vocab, y);
        f = left_of(tr, dr, taken_of<64>(a, (uint32_t)row, k), it);
        double left[VER_N];
        f.of(x, y, left);
        const double sum = wg_sum(total(left), sm);
        // the last workgroup of the request draws
        if (tid == 0) {
            // (the sum goes past the L2s, as the one that draws reads it, and has arrived before this workgroup counts itself;
            // a fence would write the whole L2 back: 3 to 10 us where 1024 workgroups do so)
            __hip_atomic_store(a.left + (uint64_t)s * a.nc + part, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            sm_last = __hip_atomic_fetch_add(a.done + s, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.nc - 1;
        }
        __syncthreads();
        if (!sm_last) return;
        double all = 0;
        for (uint32_t c = tid; c < a.nc; c += VER_T) {
            sums[c] = __hip_atomic_load(a.left + (uint64_t)s * a.nc + c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            all += sums[c];
        }
        plain = !(wg_sum(all, sm) > 0);                               // (nothing is left of p: p itself)
    }
    uint32_t next = FLH_KV_NONE;
    if (greedy) next = tr.m == -INFINITY ? FLH_KV_NONE : tr.at;
    else if (tr.m != -INFINITY) {
        __syncthreads();
        uint32_t cut = p.draft ? 0 : k;                               // tokens that are taken out
        // a chunk's weights in the order of the tokens, 16 a thread
        float x[VER_N];
        double ew[VER_N];
        auto chunk = [&](uint32_t c) {
            Chunk<T, true> xc, yc;
            xc.load(xr, c, p.vocab);
            if (!plain) yc.load(yr, c, p.vocab);
            xc.get(c, p.vocab, x);
            if (plain) {
#pragma unroll
                for (int i = 0; i < VER_N; i += 4) {
                    const float x4[4] = {x[i], x[i + 1], x[i + 2], x[i + 3]};
                    double g[4];
                    f.p.template of<4>(x4, g);
#pragma unroll
                    for (int j = 0; j < 4; ++j) ew[i + j] = g[j];
                }
            } else {
                float y[VER_N];
                yc.get(c, p.vocab, y);
                f.of(x, y, ew);
            }
            for (uint32_t g = 0; g < cut; ++g) {
#pragma unroll
                for (int i = 0; i < VER_N; ++i) ew[i] = xc.token(c, p.vocab, i) == gone[g] ? 0.0 : ew[i];
            }
        };
        for (;;) {
            if (plain) {
                for (uint32_t c = tid; c < a.nc; c += VER_T) {
                    const VerPart q = a.tp[row * a.nc + c];
                    sums[c] = q.z * f.p.of(q.m);
                }
                __syncthreads();
                // chunks that lose tokens: what goes is taken off, or, where little is left (the difference would have
                // lost digits), the rest is summed
                if (tid < cut && gone[tid] != NO_ROW) {
                    const uint32_t c = gone[tid] / VER_CH;
                    bool first = true;
                    double off = 0;
                    for (uint32_t g = 0; g < cut; ++g) {
                        const bool here = gone[g] / VER_CH == c;
                        first = first && !(here && g < tid);
                        if (here) off += gone_e[g];
                    }
                    if (first && off < 0.9375 * sums[c]) sums[c] -= off;
                    else if (first) again[atomicAdd(&n_again, 1u)] = c;
                }
                __syncthreads();
                for (uint32_t g = 0; g < (cut ? n_again : 0); ++g) {
                    chunk(again[g]);
                    const double v = wg_sum(total(ew), sm);
                    if (tid == 0) sums[again[g]] = v;
                }
                __syncthreads();
            }
            if (tid < 64) {                                           // the chunk, by one wave
                double all = 0;
                for (uint32_t c = tid; c < a.nc; c += 64) all += sums[c];
                const double want = u_next * group_sum(all);
                double before = 0, most_before = 0;
                uint32_t pick = NO_ROW, most = NO_ROW;
                for (uint32_t c0 = 0; c0 < a.nc && pick == NO_ROW; c0 += 64) {
                    const uint32_t c = c0 + tid;
                    const double v = c < a.nc ? sums[c] : 0.0;
                    const double in = wave_scan(v);
                    const uint64_t hit = __ballot(before + in > want && v > 0), some = __ballot(v > 0);
                    const int l = hit ? __builtin_ctzll(hit) : some ? 63 - __builtin_clzll(some) : 0;
                    const double at = before + lane_at(in - v, __builtin_amdgcn_readfirstlane(l));
                    if (hit) {
                        pick = c0 + l;
                        before = at;
                    } else {
                        if (some) { most = c0 + l; most_before = at; }
                        before += lane_at(in, 63);
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
            const double v = total(ew);
            double in = wave_scan(v);
            if ((tid & 63) == 63) sm[tid >> 6] = in;
            __syncthreads();
            for (uint32_t i = 0; i < tid >> 6; ++i) in += sm[i];
            // the first token whose sum passes the number; none (rounding): the last one with weight
            uint32_t hit = NO_ROW, last = NO_ROW;                     // (the last one as NO_ROW - 1 - token)
            float hit_x = 0, last_x = 0;
            double at = in - v;
#pragma unroll
            for (int i = 0; i < VER_N; ++i) {
                at += ew[i];
                const uint32_t t = Chunk<T, true>::token(c, p.vocab, i);
                const bool some = ew[i] > 0, first = some && hit == NO_ROW && at > want;
                last = some ? NO_ROW - 1 - t : last;
                last_x = some ? x[i] : last_x;
                hit = first ? t : hit;
                hit_x = first ? x[i] : hit_x;
            }
            const uint32_t h = group_min(hit), l = group_min(last);
            if ((tid & 63) == 0) {
                again[tid >> 6] = h;
                again[4 + (tid >> 6)] = l;
            }
            __syncthreads();
            const uint32_t hits = min(min(again[0], again[1]), min(again[2], again[3]));
            const uint32_t lasts = min(min(again[4], again[5]), min(again[6], again[7]));
            next = hits != NO_ROW ? hits : NO_ROW - 1 - lasts;
            if (hits != NO_ROW ? hit == hits : last == lasts) sm_x = hits != NO_ROW ? hit_x : last_x;   // (a thread's)
            __syncthreads();
        }
    }
    for (uint32_t j = tid; j < p.path_stride; j += VER_T) {
        p.path[out + j] = j < len ? w.path[j] : FLH_KV_NONE;
        if (!p.logp) continue;
        // p of the row at the token behind it
        const bool here = j + 1 == len;
        const double v = j >= len ? 1.0 : here ? tr.z : w.pc[w.path[min(j + 1, len - 1)]];
        const double lg = log(v);
        p.logp[out + j] = greedy || (here && next == FLH_KV_NONE) ? 0.f : here ? (float)(((double)sm_x - f.p.m) * it - lg) : (float)lg;
    }
    if (tid == 0) {
        p.next[s] = next;
        p.n_path[s] = len;
        if (p.len) p.len[s] = p.kv_len[s] - rows + len;
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
        a.meta = (VerMeta *)take((uint64_t)p.n_tok * sizeof(VerMeta));
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
    if (a.p.n_tok) {
        hipLaunchKernelGGL(k_verify_sums<T>, dim3(a.p.n_tok * (a.p.draft ? 2 : 1) * a.nc), dim3(64 * SUM_W), 0, s, a);
        if (int rc = hip_check(hipGetLastError(), "k_verify_sums launch")) return rc;
        for (uint32_t i = 1; i <= a.rounds; ++i) {
            hipLaunchKernelGGL(k_verify_rest<T>, dim3(a.p.n_tok * a.nc), dim3(VER_T), 0, s, a, i);
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
