// flh_attn.h -- device building blocks of the attention kernels
// (flh_attn_dec.hip, flh_attn_pre.hip, flh_attn.hip): how the work is dealt to
// workgroups, the DMA of keys and values into LDS, matrix-core wrappers.
//
// Rows and strips.  The query heads of one kv head read the same keys, so they
// are rows of one matrix: row r of request s and kv head h is token r / group,
// head h*group + r % group.  A strip is M consecutive rows.
//
// The line of work.  (request, strip, kv head, tile of KT keys that some row of
// the strip sees), in this order, is one line of U units; workgroup w of Ge
// takes units [w*U/Ge, (w+1)*U/Ge).  Lengths are on the device only, so every
// wave walks them itself (64 requests at a time, lane per request): no launch
// plans another one's grid, and a captured launch takes any lengths.  Ragged
// batches, causal strips and few long requests come out even the same way.  An
// item (request, strip, kv head) that lies across a border is worked on by
// several workgroups, which leave unscaled sums in the workspace; k_attn_join
// adds them up in line order.  Every strip has at least one unit, so
// rows that see nothing are written too.
#pragma once
#include "flh_common.h"
#include "flh_internal.h"

namespace flh {

template <typename T> struct VecOf {
    typedef T v8 __attribute__((ext_vector_type(8)));
    typedef T v4 __attribute__((ext_vector_type(4)));
};
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mma16(VecOf<_Float16>::v8 a, VecOf<_Float16>::v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(VecOf<__bf16>::v8 a, VecOf<__bf16>::v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma32(VecOf<_Float16>::v8 a, VecOf<_Float16>::v8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma32(VecOf<__bf16>::v8 a, VecOf<__bf16>::v8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// 16-bit terms that an fp32 value is split into for the matrix cores: two f16
// (11 + 11 bits) or three bf16 (8 + 8 + 8); 16-bit activations take one.
template <typename AT, typename T> constexpr int split_terms() {
    return !__is_same(AT, float) ? 1 : __is_same(T, _Float16) ? 2 : 3;
}
template <typename T, int NS> __device__ __forceinline__ void split(float x, T (&o)[NS]) {
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        o[i] = (T)x;
        x -= (float)o[i];
    }
}
// The weights exp2(score - max) are made 2^14 times larger for f16 terms, so that
// small ones do not become subnormal there; the sum has the same factor.  (A
// factor, not 14 more in the exponent: that would cost the largest weights, whose
// exponent is near 0, three bits.)
template <typename T> constexpr float weight_unit() { return __is_same(T, _Float16) ? 0x1p14f : 1.f; }

// ---------------------------------------------------------------- the line --
struct AttnItem {
    uint32_t seq, strip, kvh;
    uint32_t r0, n;                     // first row in q / out, tokens of the request
    int32_t p0;                         // position of its first row's token
    int32_t cap;                        // keys with a table entry
    int32_t lo, hi;                     // keys that some row of the strip sees
    uint32_t u0, tiles;                 // first unit of the item, units
};

template <int M, int KT> struct AttnWalk {
    const AttnArgs & a;
    const uint32_t lane;
    uint32_t base = 0, line0 = 0, all = 0;                            // this chunk of 64 requests: first one, first unit, units
    uint32_t n = 0, r0 = 0, cost = 0, excl = 0;                       // the lane's request
    int32_t p0 = 0, cap = 0;
    __device__ AttnWalk(const AttnArgs & args, uint32_t l) : a(args), lane(l) {}

    __device__ static uint32_t scan(uint32_t v, uint32_t lane) {      // inclusive, over the wave
#pragma unroll
        for (uint32_t d = 1; d < 64; d <<= 1) {
            const uint32_t o = __shfl_up(v, d);
            if (lane >= d) v += o;
        }
        return v;
    }
    // keys that strip i of a request of n tokens sees, and its units
    __device__ uint32_t span(uint32_t n_, int32_t p, int32_t c, uint32_t i, int32_t & lo, int32_t & hi) const {
        hi = c;
        lo = 0;
        if (a.causal) {
            const uint32_t t1 = min(n_ - 1, ((i + 1) * M - 1) / a.group);
            hi = max(0, min((int64_t)c, (int64_t)p + t1 + 1));
            if (a.window) {
                const uint32_t t0 = i * M / a.group;
                lo = min((int64_t)hi, max((int64_t)0, (int64_t)p + t0 + 1 - a.window));
            }
        }
        return hi > lo ? (uint32_t)((hi + KT - 1) / KT - lo / KT) : 1u;
    }
    __device__ static uint32_t strips(uint32_t n_, uint32_t group) { return (n_ * group + M - 1) / M; }

    __device__ void load(uint32_t b) {
        base = b;
        const uint32_t s = b + lane;
        n = r0 = cost = 0;
        p0 = cap = 0;
        if (s < a.n_seq) {
            const uint32_t x = min(a.q_start[s], a.n_tok), y = min(a.q_start[s + 1], a.n_tok), kv = a.kv_len[s];
            n = y > x ? y - x : 0;
            r0 = x;
            // positions and keys behind 2^30 have no table entry (see the host's check)
            const int64_t k = min((int64_t)kv, (int64_t)1 << 30);
            cap = (int32_t)min(k, (int64_t)a.table_stride << a.sh);
            p0 = (int32_t)(k - n);
        }
        const uint32_t ns = strips(n, a.group);
        int32_t lo, hi;
        if (ns == 1) cost = span(n, p0, cap, 0, lo, hi);
        uint64_t many = __ballot(ns > 1);
        while (many) {                                                // requests of many strips, lane per strip
            const int l = __builtin_ctzll(many);
            many &= many - 1;
            const uint32_t bn = __builtin_amdgcn_readlane(n, l), bs = __builtin_amdgcn_readlane(ns, l);
            const int32_t bp = __builtin_amdgcn_readlane(p0, l), bc = __builtin_amdgcn_readlane(cap, l);
            uint32_t c = 0;
            for (uint32_t i = lane; i < bs; i += 64) c += span(bn, bp, bc, i, lo, hi);
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) c += __shfl_xor(c, d);
            if (lane == (uint32_t)l) cost = c;
        }
        cost *= a.n_kv;
        const uint32_t inc = scan(cost, lane);
        excl = inc - cost;
        all = __builtin_amdgcn_readlane(inc, 63);
    }
    // units in all; leaves the walk at the first request
    __device__ uint32_t total() {
        uint32_t u = 0;
        for (uint32_t b = 0; b < a.n_seq; b += 64) {
            load(b);
            u += all;
        }
        line0 = 0;
        if (a.n_seq > 64) load(0);
        return u;
    }
    // the item of unit u (< total(), not before the chunk that the walk stands at)
    __device__ void find(uint32_t u, AttnItem & it) {
        while (u - line0 >= all) {
            line0 += all;
            load(base + 64);
        }
        uint32_t x = u - line0;
        const int l = 63 - __builtin_clzll(__ballot(excl <= x));      // (requests of no units share the next one's excl)
        it.seq = base + l;
        it.n = __builtin_amdgcn_readlane(n, l);
        it.r0 = __builtin_amdgcn_readlane(r0, l);
        it.p0 = __builtin_amdgcn_readlane(p0, l);
        it.cap = __builtin_amdgcn_readlane(cap, l);
        x -= __builtin_amdgcn_readlane(excl, l);
        const uint32_t ns = strips(it.n, a.group);
        it.strip = 0;
        if (ns > 1) {
            for (uint32_t i = 0;; i += 64) {
                int32_t lo, hi;
                const uint32_t c = i + lane < ns ? span(it.n, it.p0, it.cap, i + lane, lo, hi) * a.n_kv : 0u;
                const uint32_t inc = scan(c, lane), sum = __builtin_amdgcn_readlane(inc, 63);
                if (x >= sum && i + 64 < ns) {
                    x -= sum;
                    continue;
                }
                const int k = 63 - __builtin_clzll(__ballot(inc - c <= x && c));
                it.strip = i + k;
                x -= __builtin_amdgcn_readlane(inc - c, k);
                break;
            }
        }
        it.tiles = span(it.n, it.p0, it.cap, it.strip, it.lo, it.hi);
        it.kvh = x / it.tiles;
        it.u0 = u - x % it.tiles;
    }
};
// workgroups that share U units (at least min_units each), and their borders
__device__ __forceinline__ uint32_t attn_wgs(uint32_t U, uint32_t G, uint32_t min_units) {
    return max(1u, min(G, U / min_units));
}
__device__ __forceinline__ uint32_t attn_border(uint32_t w, uint32_t U, uint32_t Ge) {
    const uint32_t q = U / Ge, r = U % Ge;
    return w * q + min(w, r);
}

// ------------------------------------------------------------------ DMA --
// HBM -> LDS without registers: 16 (4) bytes a lane, lane l's at lds + 16 (4) * l.
// In asm, so that the compiler does not know of them: it would wait for all of
// them before every LDS read.  Whoever reads the data waits itself (wait_vm); the
// compiler's own loads beside them are waited for too long at worst.  (m0, the
// LDS base, is set each time; nothing else in these kernels uses it.)
__device__ __forceinline__ void dma16(const void * src, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(src) : "memory");
}
__device__ __forceinline__ void dma4(const void * src, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(lds), "v"(src) : "memory");
}
template <int N> __device__ __forceinline__ void wait_vm() {
    static_assert(N >= 0 && N < 64, "vmcnt has 6 bits");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint32_t lds_at(const void * p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void *)p;
}

// what a DMA reads in the place of keys that are not there
static __device__ __attribute__((aligned(16))) uint32_t g_attn_zero[4];

// 16-byte pieces of a row lie in LDS at piece ^ swz(row), so that a column of
// pieces (what a matrix-core operand reads of 16 or 32 rows) spreads over the banks
template <int D> __device__ __forceinline__ uint32_t swz(uint32_t row) { return row & (D % 128 == 0 ? 15u : 7u); }

template <typename T> __device__ __forceinline__ float load_f(const T * p) {
    T v;
    __builtin_memcpy(&v, p, sizeof v);
    return (float)v;
}
// four values as AT, at any element alignment
template <typename AT> __device__ __forceinline__ void store4(AT * p, float a, float b, float c, float d) {
    const typename VecOf<AT>::v4 v = {(AT)a, (AT)b, (AT)c, (AT)d};
    __builtin_memcpy(p, &v, sizeof v);
}
__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u; }

// Values that are no numbers.  0 * inf is NaN, so a weight of 0 (a key that a
// row does not see, or the vanished low term of a split weight) would carry an
// infinite value into the row.  The kernels do not look at the values; a piece
// whose sums come out not finite is done once more with this: the finite
// values go through the product, and for the others (1 where the class holds, 0
// elsewhere) a product with the row's visible keys (1 or 0) tells whether the
// row gets one.
template <typename T> struct ValueClass {
    u16x8 fin, pos, neg, nan;
    __device__ explicit ValueClass(typename VecOf<T>::v8 v) {
        const u16x8 b = __builtin_bit_cast(u16x8, v);
        const uint16_t E = __is_same(T, _Float16) ? 0x7C00 : 0x7F80, one = __is_same(T, _Float16) ? 0x3C00 : 0x3F80;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint16_t m = b[i] & 0x7FFF;
            fin[i] = m < E ? b[i] : (uint16_t)0;
            pos[i] = b[i] == E ? one : (uint16_t)0;
            neg[i] = m == E && b[i] != E ? one : (uint16_t)0;
            nan[i] = m > E ? one : (uint16_t)0;
        }
    }
};
__device__ __forceinline__ float odd_value(float pos, float neg, float nan) {
    const float p = pos > 0.f ? INFINITY : 0.f, q = neg > 0.f ? -INFINITY : 0.f;
    return nan > 0.f ? NAN : p + q;
}

// The plan of a launch, from host-known arguments.
struct AttnPlan {
    uint32_t grid, m, dv, min_units;
    size_t ws;
};
enum { ATTN_DIMS = 4 };
// the smallest compiled (d_k, d_v) that holds both: 0: 64 / 64, 1: 128 / 128, 2: 192 / 128, 3: 256 / 256
inline int attn_dims(const AttnArgs & a) {
    return a.dk <= 64 && a.dv <= 64 ? 0 : a.dk <= 128 && a.dv <= 128 ? 1 : a.dk <= 192 && a.dv <= 128 ? 2 : 3;
}
AttnPlan attn_dec_plan(const AttnArgs & a);
AttnPlan attn_pre_plan(const AttnArgs & a);
int launch_attn_dec(const AttnArgs & a, uint32_t dtype, uint32_t cache_dtype, hipStream_t s);
int launch_attn_pre(const AttnArgs & a, uint32_t dtype, uint32_t cache_dtype, hipStream_t s);

// Sums of the workgroups that share an item, added up: block (w, y) looks whether
// the border between workgroups w - 1 and w is the first one inside an item; a
// wave takes every fourth row of the blocks' share and adds the parts in order.
// Parts: [2 * workgroup + (1: the item begins in it)][M][DV] sums, then [M] maxima,
// [M] weights.
template <typename AT, int M, int KT, int DV>
__global__ __launch_bounds__(256) void k_attn_join(AttnArgs a) {
    const uint32_t lane = threadIdx.x & 63, w = blockIdx.x + 1;
    AttnWalk<M, KT> walk(a, lane);
    const uint32_t U = walk.total(), Ge = attn_wgs(U, a.grid, a.min_units);
    if (w >= Ge) return;
    const uint32_t u = attn_border(w, U, Ge);
    AttnItem it;
    walk.find(u, it);
    if (u == it.u0 || attn_border(w - 1, U, Ge) > it.u0) return;
    uint32_t last = w;                                                // the last workgroup with a part
    while (last + 1 < Ge && attn_border(last + 1, U, Ge) < it.u0 + it.tiles) ++last;
    const uint32_t parts = last - w + 2, rows = min((uint32_t)M, it.n * a.group - it.strip * M);
    constexpr size_t PART = (size_t)M * (DV + 2);
    const float * ws = (const float *)a.ws;
    auto part = [&](uint32_t i) { return ws + PART * (i == 0 ? 2 * (w - 1) + 1 : 2 * (w - 1 + i)); };
    constexpr int V = DV / 64;                                        // values a lane
    for (uint32_t r = blockIdx.y * 4 + (threadIdx.x >> 6); r < rows; r += 4 * gridDim.y) {
        float top = -INFINITY;
        for (uint32_t i = lane; i < parts; i += 64) top = fmaxf(top, part(i)[(size_t)M * DV + r]);
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, xor_lane(top, d, lane));
        const float base = top == -INFINITY ? 0.f : top;
        float l = 0.f, o[V];
#pragma unroll
        for (int k = 0; k < V; ++k) o[k] = 0.f;
#pragma unroll 4
        for (uint32_t i = 0; i < parts; ++i) {
            const float * p = part(i);
            const float f = __builtin_amdgcn_exp2f(p[(size_t)M * DV + r] - base);
            l = fmaf(f, p[(size_t)M * (DV + 1) + r], l);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float v = p[(size_t)r * DV + lane * V + k];
                o[k] = f == 0.f ? o[k] : fmaf(f, v, o[k]);            // (a part that sees nothing)
            }
        }
        const uint32_t row = it.strip * M + r, tok = it.r0 + row / a.group, head = it.kvh * a.group + row % a.group;
        AT * out = (AT *)a.out + tok * a.o_tok + head * a.o_head;
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (lane * V + k < a.dv) out[lane * V + k] = (AT)(l == 0.f ? 0.f : o[k] / l);
    }
}

}  // namespace flh
