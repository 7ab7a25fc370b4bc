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
// over f16 (two terms, twice the products) 626 us for 5 ragged chunks (812 TFLOP/s of products).  32 rows a wave and two
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
template <int DK, int DV> struct PreShape {
    static constexpr int W = 4;                                       // waves
    static constexpr int M = 32 * W, KT = 64, NST = 2;
    static constexpr int STAGE = KT * (DK + DV) * 2;
    // a wave's page numbers of 4 tiles, 16 keys each; row addresses of 8 tiles' keys, K and V
    static constexpr int TAB = 256 + 2 * 1024;
    static constexpr int WALK = 6 * 256;                              // AttnWalk::Chunk
    static constexpr size_t LDS = (size_t)NST * STAGE + W * (TAB + WALK) + 128;
};
template <int DK, int DV> constexpr int pre_threads = 64 * PreShape<DK, DV>::W;
// waves per SIMD that the registers are cut for, and so workgroups per CU: the grid is what
// runs at once, else some workgroups of even shares start when others are done
constexpr int pre_waves(bool split, int dk, int dv) { return dk + dv <= (split ? 128 : 256) ? 2 : 1; }

template <typename AT, typename T, int DK, int DV>
__global__ __launch_bounds__((pre_threads<DK, DV>), pre_waves(split_terms<AT, T>() > 1, DK, DV)) void k_attn_pre(AttnArgs a) {
    typedef PreShape<DK, DV> P;
    typedef typename VecOf<T>::v8 v8;
    constexpr int W = P::W, KT = P::KT, NST = P::NST, M = P::M, NS = split_terms<AT, T>();
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
    // keys of 8 tiles that have a page and that a row of the strip sees: a bit each
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
    typedef typename AttnWalk<M, KT, PRE_ITEM>::Chunk Chunk;
    static_assert(sizeof(Chunk) == P::WALK, "chunk");
    AttnWalk<M, KT, PRE_ITEM> walk(a, *(Chunk *)(sm + NST * P::STAGE + W * P::TAB + 128 + wave * P::WALK));
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
        const int32_t rhi = key_hi(a, it, tok), rlo = key_lo(a, it, tok);
        const uint32_t first = it.strip * M + 32 * wave;              // the wave's rows
        const bool here = first < rows;
        const int32_t tf = (int32_t)(first / a.group), tl = (int32_t)min(it.n - 1, (first + 31) / a.group);
        const int32_t all_lo = win ? it.p0 + tl + 1 - win : 0, all_hi = a.causal ? min(it.cap, it.p0 + tf + 1) : it.cap;

        const uint64_t zero = (uint64_t)(uintptr_t)g_attn_zero;
        const uint32_t * tab = a.table + (uint64_t)it.seq * a.table_stride;
        // The rows of four tiles are found together, 16 keys of each by the wave that brings
        // them (lane l: key l % 16 of tile 4 g + l / 16).
        auto key_of = [&](uint32_t g) { return key0 + (int32_t)((4 * g + (lane >> 4)) * KT + 16 * wave + l16); };
        auto issue_tab = [&](uint32_t g) {                            // page numbers
            const uint32_t pg = (uint32_t)min(key_of(g), max(it.cap - 1, 0)) >> a.sh;
            dma4(it.cap > 0 ? (uint64_t)(uintptr_t)(tab + pg) : zero, tab_at);
        };
        issue_tab(0);                                                 // (they arrive with the queries)

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
            const uint32_t own = *(const uint32_t *)(tabs + 4 * lane), tok = (uint32_t)key & a.pmask;
            const bool in = (key >= it.lo) & (key < it.hi) & (own < a.n_pages);
            uint64_t * rows_of = (uint64_t *)(tabs + 256) + 64 * (g & 1) + lane;
            const uint64_t kr = fresh(row_at(kb, own, a.k_page, tok, a.k_tok)), vr = fresh(row_at(vb, own, a.v_page, tok, a.v_tok));
            rows_of[0] = in ? kr : zero;
            rows_of[128] = in ? vr : zero;
            // (the 16 lanes of a tile write the same)
            ((uint16_t *)(sm_live + 4 * (g & 1) + (lane >> 4)))[wave] = (uint16_t)(__ballot(in) >> (lane & 48));
        };
        auto live = [&](uint32_t t) -> uint64_t {                     // of tile t
            const uint64_t v = sm_live[t & 7];
            return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)v);
        };
        // this wave's part of tile t's rows
        DmaRows<DK, false, NK> dk;
        DmaRows<DV, true, NV> dv;
        auto read_k = [&](uint32_t t) { dk.read(tab_at + 256 + 128 * (t & 7), fresh(lane)); };
        auto read_v = [&](uint32_t t) { dv.read(tab_at + 1280 + 128 * (t & 7), fresh(lane)); };
        auto issue_k = [&](uint32_t t) { dk.issue(fresh(lane), a.dk, zero, sm_at + (t & 1) * P::STAGE + 1024 * NK * wave); };
        auto issue_v = [&](uint32_t t) { dv.issue(fresh(lane), a.dv, zero, sm_at + (t & 1) * P::STAGE + KT * DK * 2 + 1024 * NV * wave); };

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
                const uint64_t see = fresh((vm & bits_of(rlo - k0, rhi - k0)) >> (4 * half));
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
            // K runs a tile ahead of V: stage t & 1 has K of tile t, then of t + 2, while V
            // of tile t is still needed.  Every wave brings its part at the begin of a round,
            // behind the barrier that tells that the round before is over, and waits
            // for it at the begin of the next.  Rows of the next four tiles are found in
            // round 1 of four, from page numbers asked for in round 0.
            wait_vm<0>();
            find_rows(0);
            read_k(0);
            read_v(0);
            issue_k(0);
            issue_v(0);
            read_k(1);
            issue_k(1);
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            uint64_t vm = live(0);
            if (here) scores(sm_at, sa);
            auto round = [&](uint32_t t, f32x16 (&s)[2], f32x16 (&nx)[2]) {
                read_k(t + 2);
                read_v(t + 1);
                const uint64_t now = vm;
                vm = live(t + 1);
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
                if (t + 2 < nt) issue_k(t + 2);
                if (t + 1 < nt) issue_v(t + 1);
                if ((t & 3) == 0 && t + 4 < nt) issue_tab(t / 4 + 1);
                auto midway = [&]() { if ((t & 3) == 1 && t + 3 < nt) find_rows(t / 4 + 1); };
                if (here) tile(key0 + (int32_t)(t * KT), now, sm_at + (t & 1) * P::STAGE, sm_at + (~t & 1) * P::STAGE, s, nx, midway);
                else midway();
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
            odd = odd || (lost & (key_hi(a, it, tok) > max(key_lo(a, it, tok), 0)));
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
template <typename AT, typename T, int DK, int DV> int go(const AttnArgs & a, hipStream_t s) {
    typedef PreShape<DK, DV> P;
    const void * k = (const void *)k_attn_pre<AT, T, DK, DV>;
    if (int rc = lds_fits(k, P::LDS, "k_attn_pre")) return rc;
    hipLaunchKernelGGL((k_attn_pre<AT, T, DK, DV>), dim3(a.grid), dim3(64 * P::W), P::LDS, s, a);
    if (int rc = hip_check(hipGetLastError(), "k_attn_pre launch")) return rc;
    hipLaunchKernelGGL((k_attn_join<AT, T, P::M, P::KT, DV, 1, PRE_ITEM>), dim3(a.grid, P::M / 16), dim3(256), 0, s, a);
    return hip_check(hipGetLastError(), "k_attn_join launch");
}
template <typename AT, typename T> int dims(const AttnArgs & a, hipStream_t s) {
    switch (attn_dims(a)) {
        case 0: return go<AT, T, 64, 64>(a, s);
        case 1: return go<AT, T, 128, 128>(a, s);
        case 2: return go<AT, T, 192, 128>(a, s);
        default: return go<AT, T, 256, 256>(a, s);
    }
}
template <int DK, int DV> void shape(AttnPlan & p, bool split) {
    static_assert(pre_waves(false, DK, DV) * PreShape<DK, DV>::LDS <= 160 * 1024, "workgroups per CU");
    p.dv = DV;
    p.m = PreShape<DK, DV>::M;
    p.grid = (uint32_t)(num_cus() * pre_waves(split, DK, DV));
}
}  // namespace

AttnPlan attn_pre_plan(const AttnArgs & a, uint32_t dtype) {
    AttnPlan p{};
    const bool split = dtype == FLH_DT_F32;
    switch (attn_dims(a)) {
        case 0: shape<64, 64>(p, split); break;
        case 1: shape<128, 128>(p, split); break;
        case 2: shape<192, 128>(p, split); break;
        default: shape<256, 256>(p, split); break;
    }
    // (64 tokens over 4096 keys: 48 us with 1 or 2, 38 with 4: fewer parts to join; over 512 keys
    // 23 us with 2, 24 with 4)
    p.min_units = 4;
    p.ws = attn_ws(p.grid, p.m, p.dv);
    return p;
}

int launch_attn_pre(const AttnArgs & a, uint32_t dtype, uint32_t cache_dtype, hipStream_t s) {
    if (dtype == FLH_DT_F32) return cache_dtype == FLH_DT_F16 ? dims<float, _Float16>(a, s) : dims<float, __bf16>(a, s);
    return dtype == FLH_DT_F16 ? dims<_Float16, _Float16>(a, s) : dims<__bf16, __bf16>(a, s);
}

}  // namespace flh
