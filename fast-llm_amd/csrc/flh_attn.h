// flh_attn.h -- device building blocks of the attention kernels
// (flh_attn_dec.hip, flh_attn_pre.hip, flh_attn.hip): how the work is dealt to
// workgroups, the DMA of keys and values into LDS, matrix-core wrappers.
//
// Rows and strips.  The query heads of one kv head read the same keys, so they
// are rows of one matrix: row r of request s and kv head h is token r / group,
// head h*group + r % group.  A strip is M consecutive rows.
//
// The line of work.  (request, kv head, strip, tile of KT keys that some row of
// the strip sees), in this order, is one line of U units; workgroup w of Ge
// takes units [w*U/Ge, (w+1)*U/Ge).  Lengths are on the device only, so every
// wave walks them itself (64 requests at a time, lane per request): no launch
// plans another one's grid, and a captured launch takes any lengths.  Ragged
// batches, causal strips and few long requests come out even the same way.  An
// item (request, strip, kv head) that lies across a border is worked on by
// several workgroups, which leave unscaled sums in the workspace; k_attn_join
// adds them up in line order.  Every strip has at least one unit, so
// rows that see nothing are written too.  An item's tiles stand behind C units
// with nothing in them, the cost of its begin and end in tiles: a workgroup of many
// short items gets as much time as one of a few long ones (a border among them
// stands for the item's begin).
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
// (11 + 11 bits) or three bf16 (8 + 8 + 8); 16-bit activations take one (their weights two
// in the kernel for few rows).
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
// The same for two values (one conversion for both; the rest is exact)
template <typename T, int NS> __device__ __forceinline__ void split(float x, float y, T (&o)[NS][2]) {
    typedef T t2 __attribute__((ext_vector_type(2)));
    typedef float f2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const t2 h = __builtin_convertvector(f2{x, y}, t2);
        o[i][0] = h[0];
        o[i][1] = h[1];
        x -= (float)h[0];
        y -= (float)h[1];
    }
}
// The weights exp2(score - max) are made 2^7 times larger for f16 terms, so that
// small ones do not become subnormal there; the sum has the same factor.  f16's smallest step,
// 2^-24, is then 2^-31 of a weight of 1: weights are right to 2^-32 of the row's largest,
// and n of them that are all far below it to n times that.  (A
// factor, not 7 more in the exponent: that would cost the largest weights, whose
// exponent is near 0, their last bits.)
template <typename T> constexpr float weight_unit() { return __is_same(T, _Float16) ? 0x1p7f : 1.f; }
// The running maximum moves (and the sums are rescaled) only when a score passes
// it by more than this, in powers of two: a weight is below 2^8, 2^15 with the unit,
// which f16 holds, and the sums' precision does not depend on it.
constexpr float MAX_SLACK = 8.f;

// A value that the compiler takes for a new one: what is computed from it is
// computed where it stands (a few instructions a tile), not kept in registers
// around the loop over the tiles.
__device__ __forceinline__ uint32_t fresh(uint32_t v) {
    asm volatile("" : "+v"(v));
    return v;
}
// The same for what a branch computes with: the compiler cannot move it in
// front of the branch and select afterwards, which it likes to do with register
// arithmetic that the branch is there to save.
__device__ __forceinline__ float fresh(float v) {
    asm volatile("" : "+v"(v));
    return v;
}
__device__ __forceinline__ uint64_t fresh(uint64_t v) {
    asm volatile("" : "+v"(v));
    return v;
}
// ---------------------------------------------------------------- the line --
struct AttnItem {
    uint32_t seq, strip, kvh;
    uint32_t r0, n;                     // first row in q / out, tokens of the request
    int32_t p0;                         // position of its first row's token
    int32_t cap;                        // keys with a table entry
    int32_t lo, hi;                     // keys that some row of the strip sees
    uint32_t u0, tiles;                 // first unit of the item, tiles (units: C more)
};
// keys [lo, hi) that a token of the item's request sees (any lo; none where hi <= lo or hi <= 0).
// TR, the tokens are a tree: the cached ones in front of it among them; which of the tree's own keys,
// p0 and behind, a token sees is in its bits (tree_bits).
template <bool TR> using ArgsOf = std::conditional_t<TR, AttnTreeArgs, AttnArgs>;
template <bool TR> __device__ __forceinline__ int32_t key_hi(const ArgsOf<TR> & a, const AttnItem & it, uint32_t tok) {
    if constexpr (TR) return min(it.cap, it.p0);
    return a.causal ? min(it.cap, it.p0 + (int32_t)tok + 1) : it.cap;
}
template <bool TR> __device__ __forceinline__ int32_t key_lo(const ArgsOf<TR> & a, const AttnItem & it, uint32_t tok) {
    // (a token's depth is below the request's tokens, whatever the array says)
    if constexpr (TR) tok = a.window ? min(a.tree_depth[it.r0 + min(tok, it.n - 1)], it.n - 1) : 0u;
    return a.window ? it.p0 + (int32_t)tok + 1 - (int32_t)min(a.window, 1u << 30) : 0;
}
// Bits of the 32 keys from k0 on that a token of the item's request sees in its tree (k0 below
// 2^30; the words from the token's row of the mask).  Words that are not there are zeros: loads
// of a clamped place and selects, no branch.
__device__ __forceinline__ uint32_t tree_bits(const AttnTreeArgs & a, const AttnItem & it, uint32_t tok, int32_t k0) {
    const uint32_t * row = a.tree_mask + (uint64_t)(it.r0 + min(tok, it.n - 1)) * a.tree_stride;
    const int32_t b = k0 - it.p0, w = b >> 5, last = (int32_t)a.tree_stride - 1;
    const uint32_t x = row[min(max(w, 0), last)], y = row[min(max(w + 1, 0), last)];
    const uint32_t lo = w >= 0 && w <= last ? x : 0u, hi = w >= -1 && w < last ? y : 0u;
    return __builtin_amdgcn_alignbit(hi, lo, (uint32_t)b & 31u);
}
// whether one of the keys [lo, hi) (lo >= 0, hi <= cap) has a page; by a whole wave
__device__ __forceinline__ bool any_page(const AttnArgs & a, const AttnItem & it, int32_t lo, int32_t hi) {
    const uint32_t * tab = a.table + (uint64_t)it.seq * a.table_stride;
    bool any = false;
    for (int64_t p = (lo >> a.sh) + (int64_t)(threadIdx.x & 63); __ballot(p << a.sh < hi) && !any; p += 64)
        any = __ballot(p << a.sh < hi ? tab[p] < a.n_pages : false) != 0;
    return any;
}
// tiles in front of unit x of an item
template <int C> __device__ __forceinline__ uint32_t tiles_at(uint32_t x) { return x > C ? x - C : 0u; }

template <int M, int KT, int C, bool TR = false> struct AttnWalk {
    // the wave's 64 requests at hand, in LDS (they are looked at once an item)
    struct Chunk {
        uint32_t n[64], r0[64], one[64], excl[64];                    // tokens, first row, units a kv head, units before it
        int32_t p0[64], cap[64];                                      // position of the first row, keys with a table entry
    };
    const AttnArgs & a;
    Chunk & ch;
    uint32_t base = 0, line0 = 0, all = 0;                            // the chunk's first request, first unit, units
    float about = 0.f;                                                // its units, however many
    __device__ AttnWalk(const AttnArgs & args, Chunk & c) : a(args), ch(c) {}
    template <typename V> __device__ static V get(const V & v) { return (V)__builtin_amdgcn_readfirstlane((int)v); }

    __device__ static uint32_t scan(uint32_t v, uint32_t lane) {      // inclusive, over the wave
#pragma unroll
        for (uint32_t d = 1; d < 64; d <<= 1) {
            const uint32_t o = __shfl_up(v, d);
            v += lane >= d ? o : 0u;
        }
        return v;
    }
    // keys that strip i of a request of n tokens sees, and its units
    __device__ uint32_t span(uint32_t n_, int32_t p, int32_t c, uint32_t i, int32_t & lo, int32_t & hi) const {
        hi = c;
        lo = 0;
        if constexpr (TR) {
            // (every strip: the tree's keys lie behind all of the others; a root's window begins first)
            if (a.window) lo = min((int64_t)hi, max((int64_t)0, (int64_t)p + 1 - a.window));
        } else if (a.causal) {
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

    // (No branch that only some lanes take, here and around the kernels' tiles: where
    // such branches join, the compiler has put copies of live registers in front of
    // the instruction that switches the other lanes on again, and their values were lost.)
    __device__ void load(uint32_t b) {
        const uint32_t lane = threadIdx.x & 63;
        base = b;
        const uint32_t s = min(b + lane, a.n_seq - 1);
        const bool real = b + lane < a.n_seq;
        const uint32_t first = a.q_start[s], last = a.q_start[s + 1], kv = a.kv_len[s];
        const uint32_t x = min(first, a.n_tok), y = min(last, a.n_tok), n = real && y > x ? y - x : 0;
        // positions and keys behind 2^30 have no table entry (see the host's check)
        const int32_t k = (int32_t)min(kv, 1u << 30);
        const int32_t cap = (int32_t)min((uint64_t)k, (uint64_t)a.table_stride << a.sh);
        // (rows that n_tok cuts off count for the positions of the others; a row behind
        // 2^30 in front of the first key sees nothing there either)
        const int32_t p0 = (int32_t)max((int64_t)k - (int64_t)(last > first ? last - first : 0u), -(int64_t)(1 << 30));
        const uint32_t ns = strips(n, a.group);
        int32_t lo, hi;
        uint32_t one = fresh(span(max(n, 1u), p0, cap, 0, lo, hi));
        one = ns == 1 ? one + C : 0;
        uint64_t many = __ballot(ns > 1);
        while (many) {                                                // requests of many strips, lane per strip
            const int l = __builtin_ctzll(many);
            many &= many - 1;
            const uint32_t bn = __builtin_amdgcn_readlane(n, l), bs = __builtin_amdgcn_readlane(ns, l);
            const int32_t bp = __builtin_amdgcn_readlane(p0, l), bc = __builtin_amdgcn_readlane(cap, l);
            uint32_t c = 0;
            for (uint32_t i = 0; i < bs; i += 64) {
                const uint32_t v = fresh(span(bn, bp, bc, i + lane, lo, hi));
                c += i + lane < bs ? v + C : 0u;
            }
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) c += __shfl_xor(c, d);
            one = lane == (uint32_t)l ? c : one;
        }
        const uint32_t inc = scan(one * a.n_kv, lane);
        all = __builtin_amdgcn_readlane(inc, 63);
        about = (float)one * (float)a.n_kv;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) about += __shfl_xor(about, d);
        ch.n[lane] = n;
        ch.r0[lane] = x;
        ch.one[lane] = one;
        ch.excl[lane] = inc - one * a.n_kv;
        ch.p0[lane] = p0;
        ch.cap[lane] = cap;
    }
    // units in all; leaves the walk at the first request.  0 where they pass 32 bits: the host
    // bounds what n_tok rows can give, but a q_start that does not ascend can give more.
    __device__ uint32_t total() {
        uint32_t u = 0;
        float sum = 0.f;
        for (uint32_t b = 0; b < a.n_seq; b += 64) {
            load(b);
            u += all;
            sum += about;
        }
        if (__builtin_amdgcn_readfirstlane(sum >= 4.2e9f)) return 0;
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
        const uint32_t lane = threadIdx.x & 63;
        uint32_t x = u - line0;
        const int l = 63 - __builtin_clzll(__ballot(ch.excl[lane] <= x));   // (requests of no units share the next one's excl)
        it.seq = base + l;
        it.n = get(ch.n[l]);
        it.r0 = get(ch.r0[l]);
        it.p0 = get(ch.p0[l]);
        it.cap = get(ch.cap[l]);
        x -= get(ch.excl[l]);
        const uint32_t c1 = get(ch.one[l]), ns = strips(it.n, a.group);
        it.kvh = x / c1;
        x -= it.kvh * c1;
        it.strip = 0;
        if (ns > 1) {
            for (uint32_t i = 0;; i += 64) {
                int32_t lo, hi;
                const uint32_t v = fresh(span(it.n, it.p0, it.cap, i + lane, lo, hi)), c = i + lane < ns ? v + C : 0u;
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
        it.u0 = u - x;
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
__device__ __forceinline__ void dma16(uint64_t src, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(src) : "memory");
}
__device__ __forceinline__ void dma4(uint64_t src, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(lds), "v"(src) : "memory");
}
template <int N> __device__ __forceinline__ void wait_vm() {
    static_assert(N >= 0 && N < 64, "vmcnt has 6 bits");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint32_t lds_at(const void * p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void *)p;
}

// An operand that has arrived (the compiler would wait for its load, and with it for
// every DMA, where it is first used: inside the loop)
template <typename V> __device__ __forceinline__ void arrived(V & v) {
    static_assert(sizeof(V) == 16, "four registers");
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    u4 r = __builtin_bit_cast(u4, v);
    asm volatile("" : "+v"(r));
    v = __builtin_bit_cast(V, r);
}
// base + page * stride + tok * tok_stride, in bytes (strides below 2^32)
__device__ __forceinline__ uint64_t row_at(uint64_t base, uint32_t page, uint32_t stride, uint32_t tok, uint32_t tok_stride) {
    return base + (uint64_t)page * stride + (uint64_t)tok * tok_stride;
}

// the row that a DMA reads in the place of a key that is not there
static __device__ __attribute__((aligned(16))) uint32_t g_attn_zero[128];

// A 16-byte piece of a row lies in LDS at piece ^ swz(row), so that what a
// matrix-core operand reads at once spreads over the 64 banks: for K one
// piece of 16 rows, for V (transposing reads) two or four pieces of 4 and 4 rows.
template <int D> __device__ __forceinline__ uint32_t swz_k(uint32_t row) { return D % 128 == 0 ? row & 15 : (row >> 1) & 7; }
template <int D> __device__ __forceinline__ uint32_t swz_v(uint32_t row) {
    static_assert(D == 64 || D % 128 == 0, "rows of 128 or n * 256 bytes");
    return D == 64 ? ((row & 2) << 1) | ((row >> 2) & 3) : ((row & 3) << 2) | ((row >> 2) & 3);
}
// Address of piece `at` (a constant whose low bits, the lane's, are 0) of the
// row and lane that `a` = row address + (lane's piece ^ swz) * 16 stands for: the
// swizzle works inside groups of 16 (8) pieces, to which rows are aligned.
template <int D> __device__ __forceinline__ uint32_t piece(uint32_t a, uint32_t at) {
    constexpr uint32_t G = D % 128 == 0 ? 16 : 8;
    return (a ^ (at % G * 16)) + at / G * (G * 16);
}
#define FLH_LDS(T, at) ((const __attribute__((address_space(3))) T *)(uintptr_t)(uint32_t)(at))
template <typename T> __device__ __forceinline__ typename VecOf<T>::v8 ld_row(uint32_t at) {
    return *FLH_LDS(typename VecOf<T>::v8, at);
}
// Four values of one column each, of four rows (keys): the 16 lanes of a group
// give the addresses of 4 rows x 4 pieces of 8 bytes, lane i gets column i.
template <typename T> __device__ __forceinline__ typename VecOf<T>::v4 ld_tr(uint32_t at) {
    return __builtin_bit_cast(typename VecOf<T>::v4,
                              __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(uintptr_t)at));
}

// four values as AT, at any element alignment
template <typename AT> __device__ __forceinline__ void store4(AT * p, float a, float b, float c, float d) {
    const typename VecOf<AT>::v4 v = {(AT)a, (AT)b, (AT)c, (AT)d};
    __builtin_memcpy(p, &v, sizeof v);
}
__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u; }

// A wave's N DMAs of a tile's rows (all, or from a multiple of 16 on; row numbers here
// count from there).  The addresses of the keys' rows (g_attn_zero for a key that is not
// there) stand in LDS, a key a lane wrote them; lane ln of DMA i brings one piece of row
// index(i, ln).  Pieces behind d are zeros.
template <int D, bool V, int N> struct DmaRows {
    uint64_t row[N];
    __device__ __forceinline__ static uint32_t swz(uint32_t r) { return V ? swz_v<V ? D : 64>(r) : swz_k<D>(r); }
    __device__ __forceinline__ void read(uint32_t addr, uint32_t ln) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr ((D & (D - 1)) == 0) row[i] = *FLH_LDS(uint64_t, addr + 8 * (ln / (D / 8)) + 8 * i * (512 / D));
            else row[i] = *FLH_LDS(uint64_t, addr + 8 * ((i * 64 + ln) / (D / 8)));
        }
    }
    // (the piece's place in the row: the swizzle moves bits of the row number, so the
    // lane's share and the DMA's, which is a constant, come apart)
    __device__ __forceinline__ void issue(uint32_t ln, uint32_t d, uint64_t zero, uint32_t lds) {
        uint64_t at[N];
        uint32_t e[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr ((D & (D - 1)) == 0) e[i] = ((ln % (D / 8)) ^ swz(ln / (D / 8)) ^ swz(i * (512 / D))) * 16;
            else e[i] = ((i * 64 + ln) % (D / 8) ^ swz((i * 64 + ln) / (D / 8))) * 16;
            at[i] = fresh(row[i] + e[i]);                             // (a select follows, no branch)
        }
        if (d != D) {
#pragma unroll
            for (int i = 0; i < N; ++i) at[i] = e[i] < 2 * d ? at[i] : zero;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) dma16(at[i], lds + 1024 * i);
    }
};
template <int D, bool V, int N> __device__ __forceinline__ void dma_rows(uint32_t addr, uint32_t ln, uint32_t d, uint64_t zero, uint32_t lds) {
    DmaRows<D, V, N> x;
    x.read(addr, ln);
    x.issue(ln, d, zero, lds);
}

// x where bit `at` of m is set, else -infinity
__device__ __forceinline__ float seen(float x, uint32_t m, uint32_t at) {
    const uint32_t k = (uint32_t)__builtin_amdgcn_sbfe((int)m, at, 1);
    return __uint_as_float((k & __float_as_uint(x)) | (~k & 0xFF800000u));
}
// bits [lo, hi) of 64 (any lo, hi)
__device__ __forceinline__ uint64_t bits_of(int32_t lo, int32_t hi) {
    const uint64_t a = hi >= 64 ? ~0ull : hi <= 0 ? 0ull : (1ull << hi) - 1;
    return lo <= 0 ? a : lo >= 64 ? 0ull : a & (~0ull << lo);
}
// 8 elements as they are in memory, at any element alignment
template <typename AT> struct Eight {
    AT v[8];
    // these, or zeros
    __device__ __forceinline__ void keep(bool on) {
        uint32_t w[sizeof(AT) * 2];
        __builtin_memcpy(w, v, sizeof v);
#pragma unroll
        for (uint32_t i = 0; i < sizeof(AT) * 2; ++i) w[i] = on ? w[i] : 0u;
        __builtin_memcpy(v, w, sizeof v);
    }
};
template <typename AT> __device__ __forceinline__ Eight<AT> load8(const AT * p) {
    Eight<AT> x;
    __builtin_memcpy(&x, p, sizeof x);
    return x;
}

// The plan of a launch, from host-known arguments.
struct AttnPlan {
    uint32_t grid, m, dv, min_units;
    size_t ws;
};
// the smallest compiled (d_k, d_v) that holds both: 0: 64 / 64, 1: 128 / 128, 2: 192 / 128, 3: 256 / 256
inline int attn_dims(const AttnArgs & a) {
    return a.dk <= 64 && a.dv <= 64 ? 0 : a.dk <= 128 && a.dv <= 128 ? 1 : a.dk <= 192 && a.dv <= 128 ? 2 : 3;
}
AttnPlan attn_dec_plan(const AttnTreeArgs & a);
AttnPlan attn_pre_plan(const AttnTreeArgs & a, uint32_t dtype);
// (a.tree_mask: of a tree's tokens)
int launch_attn_dec(const AttnTreeArgs & a, uint32_t dtype, uint32_t cache_dtype, hipStream_t s);
int launch_attn_pre(const AttnTreeArgs & a, uint32_t dtype, uint32_t cache_dtype, hipStream_t s);

// One row by one wave, a key a lane, in fp32 (scores from sums in 64 bits): for items whose sums are not
// finite, and rows that have keys but no weight: all their scores are -infinity, or
// finite ones passed fp32's range when they were multiplied by log2(e).  0 * inf is NaN, so in a matrix product a key
// that a row does not see (weight 0), or the vanished low term of a split weight, carries an
// infinite or NaN value into the row.  Here only the keys seen are looked at, and
// scores stay what they are, so that they are finite wherever scale q.k is.
template <typename AT, typename T, int M, bool TR> __device__ __forceinline__ void attn_row(const ArgsOf<TR> & a, const AttnItem & it, uint32_t r) {
    const uint32_t lane = threadIdx.x & 63, row = it.strip * M + r, tok = row / a.group, head = it.kvh * a.group + row % a.group;
    const AT * q = (const AT *)a.q + (it.r0 + tok) * a.q_tok + head * a.q_head;
    const int32_t old = key_hi<TR>(a, it, tok), hi = TR ? it.cap : old, lo = max(0, key_lo<TR>(a, it, tok));
    const uint64_t kb = (uint64_t)(uintptr_t)a.k + it.kvh * a.k_head, vb = (uint64_t)(uintptr_t)a.v + it.kvh * a.v_head;
    const uint32_t * tab = a.table + (uint64_t)it.seq * a.table_stride;
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    bool any = false;                                                 // a key is seen
    // (a tree behind the window of a row that is deep in it: its keys are looked at from its first on)
    for (int32_t j0 = TR ? min(lo, max(old, 0)) : lo; j0 < hi; j0 += 64) {
        const int32_t j = j0 + (int32_t)lane;
        const uint32_t pg = j < hi ? tab[(uint32_t)j >> a.sh] : FLH_KV_NONE;
        bool in = pg < a.n_pages;
        if constexpr (TR) in = in & (((j >= lo) & (j < old)) | ((tree_bits(a, it, tok, j) & 1u) != 0));
        float t = -INFINITY;
        if (in) {
            const T * k = (const T *)(uintptr_t)row_at(kb, pg, a.k_page, (uint32_t)j & a.pmask, a.k_tok);
            double dot = 0;                                           // (q.k may pass what scale q.k does not)
            for (uint32_t i = 0; i < a.dk; i += 8) {
                const Eight<T> x = load8(k + i);
                for (int e = 0; e < 8; ++e) dot = fma((double)(float)q[i + e], (double)(float)x.v[e], dot);
            }
            t = (float)(dot * (double)a.scale);
        }
        float top = t;
        for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
        const float mn = fmaxf(m, top), base = mn == -INFINITY ? 0.f : mn, al = expf(m - base), p = expf(t - base);
        float sum = p;
        for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
        l = fmaf(l, al, sum);
        m = mn;
        for (int c = 0; c < 4; ++c) o[c] *= al;
        uint64_t left = __ballot(in);
        any = any || left;
        while (left) {
            const int k = __builtin_ctzll(left);
            left &= left - 1;
            const float w = __shfl(p, k);
            const T * v = (const T *)(uintptr_t)row_at(vb, __shfl(pg, k), a.v_page, (uint32_t)(j0 + k) & a.pmask, a.v_tok);
            for (uint32_t c = 0; c < 4; ++c)
                if (64 * c + lane < a.dv) o[c] = fmaf(w, (float)v[64 * c + lane], o[c]);
        }
    }
    AT * out = (AT *)a.out + (it.r0 + tok) * a.o_tok + head * a.o_head;
    for (uint32_t c = 0; c < 4; ++c)
        if (64 * c + lane < a.dv) out[64 * c + lane] = (AT)(any ? o[c] / l : 0.f);
}

// What a launch leaves in the workspace: the parts of items that lie across a
// border, [2 * workgroup + (1: the item begins in it)][M][DV] sums, then [M]
// maxima, [M] weights; then a note for each workgroup.
struct AttnNote {
    uint32_t odd;                       // a sum of this workgroup is not finite
    uint32_t parts;                     // of the item that its first border is the first one inside (0: none)
    uint32_t seq, strip, kvh, r0, n;
    int32_t p0, cap;
    uint32_t wgs;                       // workgroups that had work (Ge; 0 if there was none)
    uint32_t pad[6];
};
template <int M, int DV> __device__ __forceinline__ float * attn_part(const AttnArgs & a, uint32_t w, bool begins) {
    return (float *)a.ws + (size_t)M * (DV + 2) * (2 * w + (begins ? 1 : 0));
}
template <int M, int DV> __device__ __forceinline__ AttnNote * attn_notes(const AttnArgs & a) {
    return (AttnNote *)((float *)a.ws + (size_t)M * (DV + 2) * 2 * a.grid);
}
inline size_t attn_ws(uint32_t grid, uint32_t m, uint32_t dv) { return (size_t)grid * (2 * m * (dv + 2) * 4 + sizeof(AttnNote)); }

// The note of workgroup w about its first item, which begins `skip` tiles before w (by a
// whole wave, every lane the same).
template <int M, int DV, int C>
__device__ __forceinline__ void attn_note(const AttnArgs & a, uint32_t w, uint32_t U, uint32_t Ge, const AttnItem & it, uint32_t skip) {
    AttnNote * n = attn_notes<M, DV>(a) + w;
    uint32_t parts = 0;
    if (skip && attn_border(w - 1, U, Ge) <= it.u0 + C) {
        uint32_t last = w;                                            // the last workgroup with a part
        while (last + 1 < Ge && attn_border(last + 1, U, Ge) < it.u0 + it.tiles + C) ++last;
        parts = last - w + 2;
        n->seq = it.seq; n->strip = it.strip; n->kvh = it.kvh; n->r0 = it.r0; n->n = it.n;
        n->p0 = it.p0; n->cap = it.cap;
    }
    n->parts = parts;
}

// Behind the main kernel.  Workgroups (w, y): the parts of w's note are added up in
// order, four rows a wave; PW waves share the parts of the same rows (a few rows of
// many parts: latency).  Rows of items with sums that are not finite, and rows that lost all their
// weight, are done by attn_row instead.  The parts' bytes bound it where there are many (18 us for those of 512
// workgroups with 128 rows of 128, up to 134 KB each; 6 for those of 256 with 32), else a launch (4 us).
template <typename AT, typename T, int M, int KT, int DV, int PW, int C, bool TR>
__global__ __launch_bounds__(256) void k_attn_join(ArgsOf<TR> a) {
    constexpr int V = DV / 64, R = 4;                                 // values a lane, rows a wave
    __shared__ float red[PW > 1 ? PW : 1][R][PW > 1 ? DV : 1];
    // Workgroups are dealt to the 8 XCDs in turn, and items that begin every 16, 32, .. workgroups would all be one XCD's,
    // whose share of the parts' bytes bounds it then (8 tokens over 4001 keys: 14 us, 6 so): within 8 neighbours w turns with
    // the bits above and with y.  Where one wave has all the rows (a single token of 4 heads), its bytes are few and its
    // own XCD's L2 has its note: one token over 4001 keys takes 13.9 us with w as it is and 14.5 turned, 2 tokens, 8 rows, 15.7 and 14.7.
    const uint32_t lane = threadIdx.x & 63, g8 = blockIdx.x >> 3;
    const bool turn = a.grid % 8 == 0 && (uint64_t)a.max_q * a.group > R;
    const uint32_t w = turn ? g8 << 3 | ((blockIdx.x + (g8 ^ g8 >> 3 ^ g8 >> 6) + blockIdx.y) & 7) : blockIdx.x;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const AttnNote * notes = attn_notes<M, DV>(a);
    // workgroups that the main kernel had no work for left no note: their number
    // is not known here, but the note of workgroup 0 tells how many had
    if (w >= notes[0].wgs) return;
    const AttnNote me = notes[w];
    const uint32_t rbase = (blockIdx.y * (4 / PW) + wave / PW) * R, pw = wave % PW;
    if (me.parts) {
        AttnItem it{};
        it.seq = me.seq; it.strip = me.strip; it.kvh = me.kvh; it.r0 = me.r0; it.n = me.n; it.p0 = me.p0; it.cap = me.cap;
        const uint32_t parts = me.parts, rows = min((uint32_t)M, it.n * a.group - it.strip * M);
        // part i of row rbase + k: its maximum, weights and values
        constexpr size_t P = (size_t)M * (DV + 2);
        const float * p0 = attn_part<M, DV>(a, w - 1, true), * p1 = attn_part<M, DV>(a, w, false);
        auto part = [&](uint32_t i) { return i == 0 ? p0 : p1 + 2 * P * (i - 1); };
        float top[R], l[R], o[R][V];
#pragma unroll
        for (int k = 0; k < R; ++k) {
            top[k] = -INFINITY;
            l[k] = 0.f;
#pragma unroll
            for (int v = 0; v < V; ++v) o[k][v] = 0.f;
        }
        uint32_t odd = 0;
        if (rbase < rows) {
            const uint32_t last_row = rows - 1;
            constexpr int Q = PW > 1 ? 8 : 2;                         // parts read at once
            float x[Q][R][V];
            auto read = [&](uint32_t i0, uint32_t n) {                // (rows behind the last one: any values)
#pragma unroll
                for (int q = 0; q < Q; ++q) {
                    const float * p = part(min(i0 + q * PW, n - 1)) + (size_t)rbase * DV + lane * V;
#pragma unroll
                    for (int k = 0; k < R; ++k)
#pragma unroll
                        for (int v = 0; v < V; ++v) x[q][k][v] = p[k * DV + v];
                }
            };
            for (uint32_t c = 0; c < parts; c += 64) {                // 64 parts, a lane each
                const uint32_t mine = min(c + lane, parts - 1), cend = min(c + 64, parts);
                float m[R], s[R], f[R];
#pragma unroll
                for (int k = 0; k < R; ++k) {
                    const float * p = part(mine) + (size_t)M * DV + min(rbase + k, last_row);
                    m[k] = p[0];
                    s[k] = p[M];
                }
                odd |= notes[w - 1 + mine].odd;
                read(c + pw, cend);
#pragma unroll
                for (int k = 0; k < R; ++k) {
                    float t = m[k];
#pragma unroll
                    for (int d = 1; d < 64; d <<= 1) t = fmaxf(t, xor_lane(t, d, lane));
                    t = fmaxf(t, top[k]);
                    const float base = t == -INFINITY ? 0.f : t, al = __builtin_amdgcn_exp2f(top[k] - base);
                    top[k] = t;
                    f[k] = c + lane < parts ? __builtin_amdgcn_exp2f(m[k] - base) : 0.f;
                    l[k] = fmaf(l[k], al, f[k] * s[k]);
#pragma unroll
                    for (int v = 0; v < V; ++v) o[k][v] *= al;
                }
                for (uint32_t i = c + pw;;) {
#pragma unroll
                    for (int q = 0; q < Q; ++q) {
                        const uint32_t j = i + q * PW;
                        if (j < cend)
#pragma unroll
                            for (int k = 0; k < R; ++k) {
                                const float g = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f[k]), j - c));
#pragma unroll
                                for (int v = 0; v < V; ++v) o[k][v] = fmaf(g, x[q][k][v], o[k][v]);
                            }
                    }
                    i += Q * PW;
                    if (i >= cend) break;
                    read(i, cend);
                }
            }
#pragma unroll
            for (int k = 0; k < R; ++k)
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) l[k] += xor_lane(l[k], d, lane);
        }
        if (rbase < rows) {
            // a bit for each row that attn_row does
            uint32_t again = 0, lost = 0;
#pragma unroll
            for (int k = 0; k < R; ++k) lost |= l[k] > 0.f ? 0u : 1u << k;   // (not a number: too)
            if (__ballot(odd != 0)) again = (1u << R) - 1;
            else
                for (uint32_t left = __builtin_amdgcn_readfirstlane(lost); left; left &= left - 1) {
                    const uint32_t k = __builtin_ctz(left), tok = (it.strip * M + min(rbase + k, rows - 1)) / a.group;
                    if (any_page(a, it, TR ? 0 : max(key_lo<TR>(a, it, tok), 0), TR ? it.cap : key_hi<TR>(a, it, tok))) again |= 1u << k;
                }
            if constexpr (PW > 1) {
#pragma unroll
                for (int k = 0; k < R; ++k)
#pragma unroll
                    for (int v = 0; v < V; ++v) red[pw][k][lane * V + v] = o[k][v];
                __syncthreads();
            }
#pragma unroll
            for (int k = 0; k < R; ++k) {
                if (rbase + k >= rows || (again >> k & 1) || (PW > 1 && k % PW != (int)pw)) continue;
                const uint32_t row = it.strip * M + rbase + k, tok = it.r0 + row / a.group, head = it.kvh * a.group + row % a.group;
                AT y[V];
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    float x = o[k][v];
                    if constexpr (PW > 1) {
                        x = red[0][k][lane * V + v];
#pragma unroll
                        for (int i = 1; i < PW; ++i) x += red[i][k][lane * V + v];
                    }
                    y[v] = (AT)(l[k] == 0.f ? 0.f : x / l[k]);
                }
                // (d_v is a multiple of 8, so of V)
                if (lane * V < a.dv) __builtin_memcpy((AT *)a.out + tok * a.o_tok + head * a.o_head + lane * V, y, sizeof y);
            }
            for (uint32_t k = PW > 1 ? pw : 0; k < R; k += PW)
                if ((again >> k & 1) && rbase + k < rows) attn_row<AT, T, M, TR>(a, it, rbase + k);
        }
    }
    if (!me.odd || pw) return;
    __shared__ typename AttnWalk<M, KT, C, TR>::Chunk chunks[4];
    AttnWalk<M, KT, C, TR> walk(a, chunks[wave]);
    const uint32_t U = walk.total(), Ge = attn_wgs(U, a.grid, a.min_units);
    const uint32_t u = attn_border(w, U, Ge), end = attn_border(w + 1, U, Ge);
    for (uint32_t x = u; x < end;) {                                  // items of workgroup w alone
        AttnItem it;
        walk.find(x, it);
        if (it.u0 + C >= u && it.u0 + it.tiles + C <= end)
            for (uint32_t r = rbase; r < min((uint32_t)M, min(rbase + R, it.n * a.group - it.strip * M)); ++r) attn_row<AT, T, M, TR>(a, it, r);
        x = it.u0 + it.tiles + C;
    }
}

}  // namespace flh
