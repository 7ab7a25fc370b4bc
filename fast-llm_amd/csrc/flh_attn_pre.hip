// flh_attn_pre.hip -- attention of many rows per kv head (prompts, chunks): the
// matrix cores and the vector instructions of the softmax are what bounds it.
#include "flh_attn.h"
#include "flh_status.h"

namespace flh {

// W waves of 32 rows each share tiles of 64 keys, which come into a ring of LDS
// stages by DMA, each wave bringing its part.  Scores are K Q^T (32x32x16
// products), so a lane holds one row's scores of 32 keys: the maximum and the sum
// are a lane's own but for one exchange with the other half of the wave, and the
// weights are, as they are, the second operand of O^T += V^T P^T (the order of the
// keys inside a product does not matter, V^T is read in the same one).  The next tile's
// scores are multiplied while this tile's weights are made (an instruction of each in
// turn), so that neither unit waits for the other.
// Roundings: with 16-bit activations a weight is rounded to the cache's type for the product
// with V (half a step of that type, as much as the rounding of the result; against the
// formula in 64 bits results are off by about 1.3 times what one rounding of them costs), while the
// sum below is of the weights as they were, in fp32.  A second term, as for few rows, would take
// 31% longer (8192 tokens in bf16: 816 us beside 621).  fp32 activations and their weights are split
// into two f16 terms, right to 2^-22 of a value, or three bf16 terms, to 2^-24; then only fp32
// accumulation rounds.
// 8192 tokens, causal, 32 / 8 heads of 128: 642 us in bf16 (857 TFLOP/s; a large library
// product reaches 1220), of which k_attn_join is 18.  The matrix cores are busy 42% of the time (at about
// 1.8 GHz under this load) and the vector instructions take as long: they hardly overlap.  fp32
// over f16 (two terms, twice the products) 603 us for 5 ragged chunks (843 TFLOP/s of products).  32 rows a wave and two
// workgroups a CU: the registers hold a wave's sums, queries and two tiles' scores (256); a
// third workgroup of narrow heads (64) would need 168 registers, spilled, and took 69 us
// instead of 63 for 8 x 20 heads over 1500 keys.
// C of the line of work.  With 0 the first workgroup of a causal prompt has most items and
// takes a third longer than the others.  us with 0 / 1 / 3 / 6, 32 / 8 heads: 8192 tokens in bf16
// 738 / 700 / 638 / 636, 2048 104 / 89 / 76 / 75; 4096 of heads of 64 166 / 146 / 130 / 133, 80 218 /
// 194 / 176 / 178, 192/128 398 / 363 / 298 / 296, 256 604 / 542 / 446 / 425; 5 chunks in fp32 over f16 659 /
// 649 / 626 / 626, over bf16 797 / 776 / 751 / 753, of heads of 256 1389 / 1332 / 1273 / 1254; 8 x 20 heads
// of 64 over 1500 keys 58 / 58 / 55 / 58; 64 requests of 40 rows over 500 keys 132 / 136 / 136 / 136.
constexpr int PRE_ITEM = 3;
static_assert(PRE_ITEM <= ATTN_ITEM, "the host's count of units");
// STAGES of the ring: with two, V of a tile comes in the round before it and K in the one before that; with three, where
// a CU's LDS holds them, both a round earlier (5 ragged chunks in fp32 over f16 603 us, 619 with two; 32 trees of 25 tokens
// over up to 8192 keys 211, 218; of heads of 192 215, 229).
template <int DK, int DV, int WAVES, int STAGES> struct PreShape {
    static constexpr int W = WAVES;
    static constexpr int M = 32 * W, KT = 64, NST = STAGES;
    static constexpr int STAGE = KT * (DK + DV) * 2;
    // A wave finds the rows of KW keys of GT tiles together, AHEAD such groups before they are read: in round FIND of a
    // group, from page numbers asked for in the round before it; K is asked for NST rounds before its own.
    static constexpr int GT = W, KW = 64 / W, AHEAD = GT < 4 ? 2 : 1, FIND = NST == 2 ? 1 : 0;
    static_assert(NST == 2 || (NST == 3 && AHEAD == 1), "rows are found in time");
    // a wave's page numbers of AHEAD groups; row addresses of two groups' keys, K and V
    static constexpr int PAGES = 256 * AHEAD, TAB = PAGES + 2 * 1024;
    static constexpr int WALK = 6 * 256;                              // AttnWalk::Chunk
    static constexpr size_t LDS = (size_t)NST * STAGE + W * (TAB + WALK) + 128;
};
// waves per SIMD that the registers are cut for, and so workgroups per CU: the grid is what
// runs at once, else some workgroups of even shares start when others are done
constexpr int pre_waves(bool split, int dk, int dv) { return dk + dv <= (split ? 128 : 256) ? 2 : 1; }
constexpr int pre_stages(bool split, int dk, int dv, int w) { return w == 4 && pre_waves(split, dk, dv) == 1 && dk + dv <= 320 ? 3 : 2; }

template <typename AT, typename T, int DK, int DV, bool TR, int WAVES>
__global__ __launch_bounds__(64 * WAVES, pre_waves(split_terms<AT, T>() > 1, DK, DV)) void k_attn_pre(ArgsOf<TR> a) {
    typedef PreShape<DK, DV, WAVES, pre_stages(split_terms<AT, T>() > 1, DK, DV, WAVES)> P;
    typedef typename VecOf<T>::v8 v8;
    constexpr int W = P::W, KT = P::KT, NST = P::NST, M = P::M, NS = split_terms<AT, T>();
    constexpr int GT = P::GT, KW = P::KW, AHEAD = P::AHEAD, FIND = P::FIND;
    constexpr int NK = DK / 8 / W, NV = DV / 8 / W;                   // DMAs of a tile, this wave's
    constexpr int DB = DV / 32;
    // Where the registers allow it: two tiles a turn of the loop, so that no scores are copied,
    // and terms of two weights at once (5 ragged chunks in fp32 over f16: 643 us without,
    // 626 with the first, 610 with both; in the forms of 256 registers either spills).
    constexpr bool ROOM = pre_waves(NS > 1, DK, DV) == 1 && DK + DV <= 320, PAIRS = ROOM && NS > 1;
    extern __shared__ __attribute__((aligned(16))) uint8_t sm[];
    const uint32_t lane = threadIdx.x & 63, l32 = lane & 31, half = lane >> 5, l16 = lane & 15;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t sm_at = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds_at(sm));
    uint8_t * tabs = sm + NST * P::STAGE + wave * P::TAB;
    const uint32_t tab_at = sm_at + NST * P::STAGE + wave * P::TAB;
    uint32_t * sm_odd = (uint32_t *)(sm + NST * P::STAGE + W * P::TAB);   // [W]
    // keys of two groups' tiles that have a page and that a row of the strip sees: a bit each
    uint64_t * sm_live = (uint64_t *)(sm_odd + 16);

    // the lane's addresses in a stage: K rows l32 (+ 32 b), pieces half (+ 2 d); V
    // rows 4 half + l16 / 4 + 8 p (+ 16 k), pieces of 16 columns by lane bit 4 (+ 4 d)
    const uint32_t k_lane = l32 * (DK * 2) + (half ^ swz_k<DK>(l32)) * 16;
    uint32_t v_lane[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        const uint32_t r = 8 * p + 4 * half + (l16 >> 2), pc = 2 * ((lane >> 4) & 1) + ((l16 >> 1) & 1);
        v_lane[p] = KT * DK * 2 + r * (DV * 2) + (pc ^ swz_v<DV>(r)) * 16 + (l16 & 1) * 8;
    }
    typedef typename AttnWalk<M, KT, PRE_ITEM, TR>::Chunk Chunk;
    static_assert(sizeof(Chunk) == P::WALK, "chunk");
    AttnWalk<M, KT, PRE_ITEM, TR> walk(a, *(Chunk *)(sm + NST * P::STAGE + W * P::TAB + 128 + wave * P::WALK));
    const uint32_t U = walk.total(), Ge = attn_wgs(U, a.grid, a.min_units);
    // neighbours on the line share keys: they go to one XCD (workgroups are dealt
    // to the 8 XCDs in turn)
    const uint32_t w = Ge == a.grid && a.grid % 8 == 0 ? (blockIdx.x & 7) * (a.grid / 8) + (blockIdx.x >> 3) : blockIdx.x;
    if (w >= Ge) return;
    uint32_t u = attn_border(w, U, Ge);
    const uint32_t first_u = u;
    const uint32_t end = attn_border(w + 1, U, Ge);
    bool odd = false;                                                 // a sum is not finite, or a row lost its weight
    while (u < end) {
        AttnItem it;
        walk.find(u, it);
        const uint32_t skip = tiles_at<PRE_ITEM>(u - it.u0), nt = tiles_at<PRE_ITEM>(min(it.tiles + PRE_ITEM, end - it.u0)) - skip;
        if (u == first_u && wave == 0) attn_note<M, DV, PRE_ITEM>(a, w, U, Ge, it, skip);
        if (nt == 0) break;                                           // (the workgroup ends among the item's empty units)
        const int32_t key0 = (int32_t)((it.lo / KT + skip) * KT);
        const bool begins = skip == 0, ends = skip + nt == it.tiles;
        const uint32_t rows = it.n * a.group, row = it.strip * M + 32 * wave + l32, tok = row / a.group;
        const uint32_t head = it.kvh * a.group + row % a.group;
        const int32_t win = (int32_t)min(a.window, 1u << 30);
        // keys that the lane's row sees; that all of the wave's rows see
        const int32_t rhi = key_hi<TR>(a, it, tok), rlo = key_lo<TR>(a, it, tok);
        const uint32_t first = it.strip * M + 32 * wave;              // the wave's rows
        const bool here = first < rows;
        const int32_t tf = (int32_t)(first / a.group), tl = (int32_t)min(it.n - 1, (first + 31) / a.group);
        // (a tree: the deepest token that there may be)
        const int32_t all_lo = win ? it.p0 + (TR ? (int32_t)it.n - 1 : tl) + 1 - win : 0;
        const int32_t all_hi = TR ? min(it.cap, it.p0) : a.causal ? min(it.cap, it.p0 + tf + 1) : it.cap;

        const uint64_t zero = (uint64_t)(uintptr_t)g_attn_zero;
        const uint32_t * tab = a.table + (uint64_t)it.seq * a.table_stride;
        // The rows of a group of GT tiles are found together, KW keys of each by the wave that brings
        // them (lane l: key l % KW of tile GT g + l / KW).
        auto key_of = [&](uint32_t g) { return key0 + (int32_t)((GT * g + lane / KW) * KT + KW * wave + lane % KW); };
        auto issue_tab = [&](uint32_t g) {                            // page numbers
            const uint32_t pg = (uint32_t)min(key_of(g), max(it.cap - 1, 0)) >> a.sh;
            dma4(it.cap > 0 ? (uint64_t)(uintptr_t)(tab + pg) : zero, tab_at + (AHEAD > 1 ? (g & 1) * 256 : 0));
        };
        issue_tab(0);
        if constexpr (AHEAD > 1) issue_tab(1);                                                 // (they arrive with the queries)

        // ---- queries: column l32, elements 16 s + 8 half ..
        v8 qf[NS][DK / 16];
        float c = a.scale == 0.f ? 1.f : a.scale * 1.4426950408889634f;   // scale * log2(e), by row
        {
            // scale 0: every score is 0.  A lane with no row or elements behind d reads the
            // first of the item instead.
            const bool real = row < rows && a.scale != 0.f;
            const AT * q = (const AT *)a.q + (it.r0 + (row < rows ? tok : 0u)) * a.q_tok + (row < rows ? head : it.kvh * a.group) * a.q_head;
            Eight<AT> x[DK / 16];
            float top = 0.f;
#pragma unroll
            for (int s = 0; s < DK / 16; ++s) {
                const uint32_t e = 16 * s + 8 * half;
                x[s] = load8(q + (e < a.dk ? e : 0u));
            }
#pragma unroll
            for (int s = 0; s < DK / 16; ++s) x[s].keep(real & (16 * s + 8 * half < a.dk));
            int ex = 0;
            if constexpr (NS == 2) {
                // f16 terms: the row's largest element to [2^13, 2^14), and back in c
#pragma unroll
                for (int s = 0; s < DK / 16; ++s)
#pragma unroll
                    for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf((float)x[s].v[j]));
                top = fmaxf(top, xor_lane(top, 32, lane));
                ex = top > 0.f && finite(top) ? 13 - ilogbf(top) : 0;
                c = fmaxf(ldexpf(c, -ex), 0x1p-126f);                 // (c * -inf below)
            }
#pragma unroll
            for (int s = 0; s < DK / 16; ++s)
                if constexpr (NS == 1) {
                    qf[0][s] = __builtin_bit_cast(v8, x[s]);
                    arrived(qf[0][s]);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        T o[NS];
                        split<T, NS>(NS == 2 ? ldexpf(x[s].v[j], ex) : (float)x[s].v[j], o);
#pragma unroll
                        for (int t = 0; t < NS; ++t) qf[t][s][j] = o[t];
                    }
                }
        }

        const uint64_t kb = (uint64_t)(uintptr_t)a.k + it.kvh * a.k_head, vb = (uint64_t)(uintptr_t)a.v + it.kvh * a.v_head;
        auto find_rows = [&](uint32_t g) {                            // from them, row addresses and live keys
            const int32_t key = key_of(g);
            const uint32_t own = *(const uint32_t *)(tabs + (AHEAD > 1 ? (g & 1) * 256 : 0) + 4 * lane), tok = (uint32_t)key & a.pmask;
            const bool in = (key >= it.lo) & (key < it.hi) & (own < a.n_pages);
            uint64_t * rows_of = (uint64_t *)(tabs + P::PAGES) + 64 * (g & 1) + lane;
            const uint64_t kr = fresh(row_at(kb, own, a.k_page, tok, a.k_tok)), vr = fresh(row_at(vb, own, a.v_page, tok, a.v_tok));
            rows_of[0] = in ? kr : zero;
            rows_of[128] = in ? vr : zero;
            // (the lanes of a tile write the same)
            typedef std::conditional_t<KW == 16, uint16_t, uint32_t> Keys;
            ((Keys *)(sm_live + GT * (g & 1) + lane / KW))[wave] = (Keys)(__ballot(in) >> (lane & ~(KW - 1)));
        };
        auto live = [&](uint32_t t) -> uint64_t {                     // of tile t
            const uint64_t v = sm_live[t & (2 * GT - 1)];
            return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)v);
        };
        // this wave's part of tile t's rows
        DmaRows<DK, false, NK> dk;
        DmaRows<DV, true, NV> dv;
        auto read_k = [&](uint32_t t) { dk.read(tab_at + P::PAGES + 8 * KW * (t & (2 * GT - 1)), fresh(lane)); };
        auto read_v = [&](uint32_t t) { dv.read(tab_at + P::PAGES + 1024 + 8 * KW * (t & (2 * GT - 1)), fresh(lane)); };
        auto issue_k = [&](uint32_t at) { dk.issue(fresh(lane), a.dk, zero, at + 1024 * NK * wave); };       // (into a stage)
        auto issue_v = [&](uint32_t at) { dv.issue(fresh(lane), a.dv, zero, at + KT * DK * 2 + 1024 * NV * wave); };

        float m, l;
        f32x16 o[DB];
        f32x16 sa[2], sb[2];                                          // scores of the tile at hand and the next
        // the tile at `at` times the queries, in steps of 16 elements
        auto scores = [&](uint32_t at, f32x16 (&x)[2]) {
            const uint32_t ka = fresh(at + k_lane);
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) x[b][i] = 0.f;
#pragma unroll
            for (int d = 0; d < DK / 16; ++d)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const v8 kf = ld_row<T>(piece<DK>(ka, 2 * d) + 32 * b * DK * 2);
#pragma unroll
                    for (int t2 = NS - 1; t2 >= 0; --t2) x[b] = mma32(kf, qf[t2][d], x[b]);
                }
        };
        // s: a tile's scores -> sums; the scores of the next one (K at `next`) are
        // multiplied meanwhile into nx; `midway` is called on the way
        auto tile = [&](int32_t k0, uint64_t vm, uint32_t at, uint32_t next, f32x16 (&s)[2], f32x16 (&nx)[2], auto && midway) {
            if (!(vm == ~0ull && k0 >= all_lo && k0 + KT <= all_hi)) {
                uint64_t may = bits_of(rlo - k0, rhi - k0);
                if constexpr (TR) {
                    if (k0 + KT > all_hi) may |= (uint64_t)tree_bits(a, it, tok, k0 + 32) << 32 | tree_bits(a, it, tok, k0);
                }
                const uint64_t see = fresh((vm & may) >> (4 * half));
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        s[b][i] = seen(s[b][i], (uint32_t)(see >> (32 * b)), 8 * (i >> 2) + (i & 3));
            }
            float top = -INFINITY;
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
            top = fmaxf(top, xor_lane(top, 32, lane));
            top *= c;
            if (__ballot(top > m + MAX_SLACK)) {
                const float mn = top > m + MAX_SLACK ? top : m, al = fresh(mn == m ? 1.f : __builtin_amdgcn_exp2f(m - mn));
                m = mn;
                l *= al;
#pragma unroll
                for (int d = 0; d < DB; ++d) o[d] *= al;
            }
            const float base = m == -INFINITY ? 0.f : m;
            // ---- the products run under the vector instructions.  The order is fixed by
            // hand (the barriers stop the compiler, which would gather the products): step i
            // of the next tile's scores (one K operand, read three steps before) with a share
            // of the weights of the first 32 keys; then V, 16 keys and up to 128 columns a
            // step, the first steps with the weights of the other 32 keys.
            float sum = 0.f;
            v8 pf[KT / 16][NS];
            // a weight in three pieces of work, which are put a step apart (the results of
            // one come late for the next)
            auto arg = [&](int e0, int e1) {
#pragma unroll
                for (int e = e0; e < e1; ++e) s[e >> 4][e & 15] = fmaf(s[e >> 4][e & 15], c, -base);
            };
            auto exps = [&](int e0, int e1) {
#pragma unroll
                for (int e = e0; e < e1; ++e) s[e >> 4][e & 15] = __builtin_amdgcn_exp2f(s[e >> 4][e & 15]);
            };
            auto pack = [&](int e0, int e1) {
#pragma unroll
                for (int e = e0; e < e1; ++e) {
                    const float p = s[e >> 4][e & 15] * weight_unit<T>();
                    sum += p;
                    if constexpr (PAIRS) {
                        if ((e & 1) == 0) continue;
                        T h[NS][2];
                        split<T, NS>(s[e >> 4][(e & 15) - 1] * weight_unit<T>(), p, h);
#pragma unroll
                        for (int t2 = 0; t2 < NS; ++t2) {
                            pf[e >> 3][t2][(e & 7) - 1] = h[t2][0];
                            pf[e >> 3][t2][e & 7] = h[t2][1];
                        }
                    } else {
                        T h[NS];
                        split<T, NS>(p, h);
#pragma unroll
                        for (int t2 = 0; t2 < NS; ++t2) pf[e >> 3][t2][e & 7] = h[t2];
                    }
                }
            };
            // step i of n of the 16 weights from e0 on
            auto weights = [&](int i, int n, int e0) {
                const int q = n - 2;
                constexpr int S = PAIRS ? 2 : 1;
                if (i < q) exps(e0 + 16 / S * i / q * S, e0 + 16 / S * (i + 1) / q * S);
                if (i >= 1 && i <= q) pack(e0 + 16 / S * (i - 1) / q * S, e0 + 16 / S * i / q * S);
            };
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) nx[b][i] = 0.f;
            constexpr int NF = DK / 8;                                // K operands of a tile
            const uint32_t ka = fresh(next + k_lane), va[2] = {fresh(at + v_lane[0]), fresh(at + v_lane[1])};
            v8 kf[4];
            auto ld_k = [&](int i) { kf[i & 3] = ld_row<T>(piece<DK>(ka, 2 * (i >> 1)) + 32 * (i & 1) * DK * 2); };
            constexpr int DC = DB < 4 ? DB : 4, VSTEPS = KT / 16 * (DB / DC);
            v8 vf[2][DC];
            auto ld_v = [&](int step) {
                const int k = step / (DB / DC), d0 = step % (DB / DC) * DC;
#pragma unroll
                for (int d = 0; d < DC; ++d)
#pragma unroll
                    for (int p = 0; p < 2; ++p) {
                        const typename VecOf<T>::v4 r4 = ld_tr<T>(piece<DV>(va[p], 4 * (d0 + d)) + 16 * k * DV * 2);
#pragma unroll
                        for (int j = 0; j < 4; ++j) vf[step & 1][d][4 * p + j] = r4[j];
                    }
            };
            // (of a SIMD's two waves the one with products goes first: 640 -> 618 us, 8192 tokens, bf16)
            __builtin_amdgcn_s_setprio(1);
            ld_k(0);
            ld_k(1);
            ld_k(2);
#pragma unroll
            for (int i = 0; i < NF; ++i) {
                __builtin_amdgcn_sched_barrier(0);
                if (i + 3 < NF) ld_k(i + 3);
                if (i + 3 == NF) ld_v(0);
#pragma unroll
                for (int t2 = NS - 1; t2 >= 0; --t2) nx[i & 1] = mma32(kf[i & 3], qf[t2][i >> 1], nx[i & 1]);
                arg(32 * i / NF, 32 * (i + 1) / NF);
                if (i) weights(i - 1, NF - 1, 0);
                if (i == NF / 2) midway();
            }
#pragma unroll
            for (int step = 0; step < VSTEPS; ++step) {
                const int k = step / (DB / DC), d0 = step % (DB / DC) * DC;
                __builtin_amdgcn_sched_barrier(0);
                if (step + 1 < VSTEPS) ld_v(step + 1);
#pragma unroll
                for (int t2 = NS - 1; t2 >= 0; --t2)
#pragma unroll
                    for (int d = 0; d < DC; ++d) {
                        __builtin_amdgcn_sched_barrier(0);
                        o[d0 + d] = mma32(vf[step & 1][d], pf[k][t2], o[d0 + d]);
                        // the first half of the steps' products carry the weights 16 .. 31
                        constexpr int H = VSTEPS / 2 * NS * DC;
                        const int i = (step * NS + (NS - 1 - t2)) * DC + d;
                        if (i < H) weights(i, H, 16);
                    }
            }
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(0);
            l += sum;
        };
        {
            m = -INFINITY;
            l = 0.f;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
            // K runs a tile ahead of V: stage t % NST has K of tile t, then of t + NST, while V
            // of tile t is still needed.  Every wave brings its part at the begin of a round,
            // behind the barrier that tells that the round before is over, and waits
            // for it at the begin of the next but NST - 2.
            wait_vm<0>();
            find_rows(0);
            if constexpr (AHEAD > 1) find_rows(1);
            if constexpr (FIND == 0) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");    // (the page numbers are read)
                issue_tab(1);
            }
            uint32_t at[NST];                                         // stages of this round's tile and those behind it
#pragma unroll
            for (int i = 0; i < NST; ++i) at[i] = sm_at + i * P::STAGE;
#pragma unroll
            for (int i = 0; i < NST; ++i) {
                read_k(i);
                if (i + 1 < NST) read_v(i);
                issue_k(at[i]);
                if (i + 1 < NST) issue_v(at[i]);
            }
            // (of three K and two V, the first two K and the first V)
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(NST == 3 ? NK + NV : 0) : "memory");
            uint64_t vm = live(0);
            if (here) scores(at[0], sa);
            auto round = [&](uint32_t t, f32x16 (&s)[2], f32x16 (&nx)[2]) {
                read_k(t + NST);
                read_v(t + NST - 1);
                const uint64_t now = vm;
                vm = live(t + 1);
                // (what the round before asked for, K of tile t + 2 and V of t + 1, may be on its way with three stages)
                if (NST == 3 && t + 2 < nt) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(NK + NV) : "memory");
                else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
                if ((t + 1) % GT == FIND && t + 1 - FIND + AHEAD * GT < nt) issue_tab((t + 1) / GT + AHEAD);
                if (t + NST < nt) issue_k(at[0]);
                if (t + NST - 1 < nt) issue_v(at[NST - 1]);
                auto midway = [&]() { if (t % GT == FIND && t - FIND + AHEAD * GT < nt) find_rows(t / GT + AHEAD); };
                if (here) tile(key0 + (int32_t)(t * KT), now, at[0], at[1], s, nx, midway);
                else midway();
                const uint32_t old = at[0];
#pragma unroll
                for (int i = 0; i + 1 < NST; ++i) at[i] = at[i + 1];
                at[NST - 1] = old;
            };
            if constexpr (ROOM) {
                for (uint32_t t = 0; t < nt; t += 2) {
                    round(t, sa, sb);
                    if (t + 1 < nt) round(t + 1, sb, sa);
                }
            } else {
                for (uint32_t t = 0; t < nt; ++t) {
                    round(t, sa, sb);
                    sa[0] = sb[0];
                    sa[1] = sb[1];
                }
            }
            wait_vm<0>();
            odd = odd || !finite(l);
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) odd = odd || !finite(o[d][i]);
        }
        l += xor_lane(l, 32, lane);
        const bool whole = begins && ends;
        // a row that has keys got no weight
        const bool lost = !(l > 0.f) & (row < rows);
        if (__ballot(lost) && whole && any_page(a, it, it.lo, it.hi))
            odd = odd || (lost & (TR || key_hi<TR>(a, it, tok) > max(key_lo<TR>(a, it, tok), 0)));
        if (row < rows) {
            if (whole) {
                AT * out = (AT *)a.out + (it.r0 + tok) * a.o_tok + head * a.o_head;
                const float f = 1.f / l;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t e = 32 * d + 8 * k + 4 * half;
                        if (e >= a.dv) continue;
                        float v[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[i] = l == 0.f ? 0.f : o[d][4 * k + i] * f;
                        store4(out + e, v[0], v[1], v[2], v[3]);
                    }
            } else {
                float * part = attn_part<M, DV>(a, w, begins);
                const uint32_t r = 32 * wave + l32;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        *(f32x4 *)(part + (size_t)r * DV + 32 * d + 8 * k + 4 * half) =
                            f32x4{o[d][4 * k], o[d][4 * k + 1], o[d][4 * k + 2], o[d][4 * k + 3]};
                if (half == 0) {
                    part[(size_t)M * DV + r] = m;
                    part[(size_t)M * (DV + 1) + r] = l;
                }
            }
        }
        u = it.u0 + PRE_ITEM + skip + nt;
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");   // the next item's stages
    }
    sm_odd[wave] = __ballot(odd) != 0;
    __syncthreads();
    if (wave == 0) {
        uint32_t f = 0;
        for (int i = 0; i < W; ++i) f |= sm_odd[i];
        AttnNote * n = attn_notes<M, DV>(a) + w;
        n->odd = f;
        n->wgs = U ? Ge : 0;
    }
}

namespace {
template <typename AT, typename T, int DK, int DV, bool TR, int W = 4> int go(const ArgsOf<TR> & a, hipStream_t s) {
    typedef PreShape<DK, DV, W, pre_stages(split_terms<AT, T>() > 1, DK, DV, W)> P;
    const void * k = (const void *)k_attn_pre<AT, T, DK, DV, TR, W>;
    if (int rc = lds_fits(k, P::LDS, "k_attn_pre")) return rc;
    hipLaunchKernelGGL((k_attn_pre<AT, T, DK, DV, TR, W>), dim3(a.grid), dim3(64 * W), P::LDS, s, a);
    if (int rc = hip_check(hipGetLastError(), "k_attn_pre launch")) return rc;
    hipLaunchKernelGGL((k_attn_join<AT, T, P::M, P::KT, DV, 1, PRE_ITEM, TR>), dim3(a.grid, P::M / 16), dim3(256), 0, s, a);
    return hip_check(hipGetLastError(), "k_attn_join launch");
}
template <typename AT, typename T, bool TR> int dims(const ArgsOf<TR> & a, hipStream_t s) {
    switch (attn_dims(a)) {
        case 0: return go<AT, T, 64, 64, TR>(a, s);
        case 1: return go<AT, T, 128, 128, TR>(a, s);
        case 2: return go<AT, T, 192, 128, TR>(a, s);
        default: return go<AT, T, 256, 256, TR>(a, s);
    }
}
// Trees in fp32, whose form has one wave a SIMD: strips of 64 rows, two waves, two workgroups on a CU, where no request has
// more rows a kv head, or most have no more (half of the waves of a strip of 128 would have no rows).  us with 128 / 64, 32
// requests of 32 to 8192 keys, 32 / 8 heads, over f16 (over bf16); rows on average, as a share of the most:
//   tokens               heads of 128              heads of 64
//   9              1     176 / 138 (213 / 151)      93 / 80 (109 / 92)     one strip of 64 each
//   1 to 20        .53   179 / 144 (213 / 157)
//   1 to 25        .52   181 / 156 (217 / 173)      94 / 91 (111 / 105)    a third have two
//   1 to 32        .52   195 / 180 (237 / 204)
//   27, 1, 1, 1    .28   181 / 146 (218 / 161)      96 / 88 (114 / 101)
//   27, 1          .52   196 / 186 (231 / 210)     104 / 111 (123 / 129)   half have two
//   17, 1          .53   178 / 170 (219 / 195)      95 / 106
//   17, 17, 1      .69   183 / 193 (216 / 217)                             two thirds
//   17, 17, 17, 1  .76   180 / 198 (220 / 221)
//   25             1     216 / 261                 119 / 152               all
// Over 65536 keys 4 of 16 tokens take 279 / 224 and 342 / 256.  So half of the requests may have two strips with heads of 128, which
// the average tells where they are spread out: up to 9/16 of the most.  With heads of 64 that gains too little: one strip
// each, by max_q.  n_tok is the rows that there may be: where a captured step has room for more than it has
// rows, the average says too much and strips stay at 128.
bool may_half(const AttnTreeArgs & a, bool split) { return a.tree_stride && split && attn_dims(a) < 2; }
bool half(const AttnTreeArgs & a, bool split) {
    const uint64_t most = (uint64_t)a.max_q * a.group;
    return may_half(a, split) &&
           (most <= 64 || (attn_dims(a) == 1 && most <= 128 && 16ull * a.n_tok * a.group <= 9 * most * a.n_seq));
}
template <typename AT, typename T> int forms(const AttnTreeArgs & a, hipStream_t s) {
    if constexpr (split_terms<AT, T>() > 1)
        if (half(a, true)) return attn_dims(a) == 0 ? go<AT, T, 64, 64, true, 2>(a, s) : go<AT, T, 128, 128, true, 2>(a, s);
    return a.tree_stride ? dims<AT, T, true>(a, s) : dims<AT, T, false>(a, s);
}
template <int DK, int DV> void shape(AttnPlan & p, bool split) {
    static_assert(pre_waves(false, DK, DV) * PreShape<DK, DV, 4, pre_stages(false, DK, DV, 4)>::LDS <= 160 * 1024, "workgroups per CU");
    static_assert(pre_waves(true, DK, DV) * PreShape<DK, DV, 4, pre_stages(true, DK, DV, 4)>::LDS <= 160 * 1024, "workgroups per CU");
    p.dv = DV;
    p.m = 128;
    p.grid = (uint32_t)(num_cus() * pre_waves(split, DK, DV));
}
}  // namespace

AttnPlan attn_pre_plan(const AttnTreeArgs & a, uint32_t dtype) {
    AttnPlan p{};
    const bool split = dtype == FLH_DT_F32;
    switch (attn_dims(a)) {
        case 0: shape<64, 64>(p, split); break;
        case 1: shape<128, 128>(p, split); break;
        case 2: shape<192, 128>(p, split); break;
        default: shape<256, 256>(p, split); break;
    }
    p.ws = attn_ws(p.grid, p.m, p.dv);
    if (may_half(a, split)) {
        static_assert(3 * PreShape<64, 64, 2, 2>::LDS <= 160 * 1024 && 2 * PreShape<128, 128, 2, 2>::LDS <= 160 * 1024, "workgroups per CU");
        const uint32_t grid = (uint32_t)num_cus() * (attn_dims(a) == 0 ? 3 : 2);
        p.ws = std::max(p.ws, attn_ws(grid, 64, p.dv));           // (the same for any number of rows)
        if (half(a, split)) {
            p.m = 64;
            p.grid = grid;
        }
    }
    // (64 tokens over 4096 keys: 48 us with 1 or 2, 38 with 4: fewer parts to join; over 512 keys
    // 23 us with 2, 24 with 4)
    p.min_units = 4;
    return p;
}

int launch_attn_pre(const AttnTreeArgs & a, uint32_t dtype, uint32_t cache_dtype, hipStream_t s) {
    if (dtype == FLH_DT_F32) return cache_dtype == FLH_DT_F16 ? forms<float, _Float16>(a, s) : forms<float, __bf16>(a, s);
    return dtype == FLH_DT_F16 ? forms<_Float16, _Float16>(a, s) : forms<__bf16, __bf16>(a, s);
}

}  // namespace flh
