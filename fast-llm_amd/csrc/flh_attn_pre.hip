// flh_attn_pre.hip -- attention of many rows per kv head (prompts, chunks): the
// matrix cores are what bounds it.
#include "flh_attn.h"
#include "flh_status.h"

namespace flh {

// W waves of 32 rows each share tiles of 64 keys, which come into a ring of LDS
// stages by DMA, each wave bringing its part.  Scores are K Q^T (32x32x16
// products), so a lane holds one row's scores of 32 keys: the maximum and the sum
// are a lane's own but for one exchange with the other half of the wave, and the
// weights are, as they are, the second operand of O^T += V^T P^T (the order of the
// keys inside a product does not matter, V^T is read in the same one).
template <int DK, int DV> struct PreShape {
    static constexpr int W = 4;                                       // waves
    static constexpr int M = 32 * W, KT = 64, NST = 2;
    static constexpr int STAGE = KT * (DK + DV) * 2;
    static constexpr int TAB = 2 * 256 + 1024;                        // a wave's page numbers of two tiles, row addresses of one
    static constexpr size_t LDS = (size_t)NST * STAGE + W * TAB + 64;
};
template <int DK, int DV> constexpr int pre_threads = 64 * PreShape<DK, DV>::W;
// waves per SIMD that the registers are cut for
template <typename AT, typename T, int DK, int DV> constexpr int pre_waves = DK + DV <= 256 && split_terms<AT, T>() == 1 ? 2 : 1;

template <typename AT, typename T, int DK, int DV>
__global__ __launch_bounds__((pre_threads<DK, DV>), (pre_waves<AT, T, DK, DV>)) void k_attn_pre(AttnArgs a) {
    typedef PreShape<DK, DV> P;
    typedef typename VecOf<T>::v8 v8;
    constexpr int W = P::W, KT = P::KT, NST = P::NST, M = P::M, NS = split_terms<AT, T>();
    constexpr int NK = DK / 8 / W, NV = DV / 8 / W, ND = NK + NV;     // DMAs of a tile, this wave's
    constexpr int DB = DV / 32;
    extern __shared__ __attribute__((aligned(16))) uint8_t sm[];
    const uint32_t lane = threadIdx.x & 63, l32 = lane & 31, half = lane >> 5, l16 = lane & 15;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t sm_at = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds_at(sm));
    uint8_t * tabs = sm + NST * P::STAGE + wave * P::TAB;
    const uint32_t tab_at = sm_at + NST * P::STAGE + wave * P::TAB;
    uint32_t * sm_odd = (uint32_t *)(sm + NST * P::STAGE + W * P::TAB);   // [W]

    // the lane's addresses in a stage: K rows l32 (+ 32 b), pieces half (+ 2 d); V
    // rows 4 half + l16 / 4 + 8 p (+ 16 k), pieces of 16 columns by lane bit 4 (+ 4 d)
    const uint32_t k_lane = l32 * (DK * 2) + (half ^ swz_k<DK>(l32)) * 16;
    uint32_t v_lane[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        const uint32_t r = 8 * p + 4 * half + (l16 >> 2), pc = 2 * ((lane >> 4) & 1) + ((l16 >> 1) & 1);
        v_lane[p] = KT * DK * 2 + r * (DV * 2) + (pc ^ swz_v<DV>(r)) * 16 + (l16 & 1) * 8;
    }
    AttnWalk<M, KT> walk(a, lane);
    const uint32_t U = walk.total(), Ge = attn_wgs(U, a.grid, a.min_units);
    // neighbours on the line share keys: they go to one XCD (workgroups are dealt
    // to the 8 XCDs in turn)
    const uint32_t w = Ge == a.grid && a.grid % 8 == 0 ? (blockIdx.x & 7) * (a.grid / 8) + (blockIdx.x >> 3) : blockIdx.x;
    if (w >= Ge) return;
    uint32_t u = attn_border(w, U, Ge);
    const uint32_t first_u = u;
    const uint32_t end = attn_border(w + 1, U, Ge);
    bool odd = false;                                                 // a sum is not finite
    while (u < end) {
        AttnItem it;
        walk.find(u, it);
        const uint32_t skip = u - it.u0, nt = min(it.tiles - skip, end - u);
        const int32_t key0 = (int32_t)((it.lo / KT + skip) * KT);
        const bool begins = skip == 0, ends = skip + nt == it.tiles;
        if (u == first_u && threadIdx.x == 0) attn_note<M, DV>(a, w, U, Ge, it, skip);
        const uint32_t rows = it.n * a.group, row = it.strip * M + 32 * wave + l32, tok = row / a.group;
        const uint32_t head = it.kvh * a.group + row % a.group;
        const int32_t win = (int32_t)min(a.window, 1u << 30);
        // keys that the lane's row sees; that a row of the wave sees; that all of them see
        const int32_t rhi = a.causal ? min(it.cap, it.p0 + (int32_t)tok + 1) : it.cap;
        const int32_t rlo = win ? it.p0 + (int32_t)tok + 1 - win : 0;
        const uint32_t first = it.strip * M + 32 * wave;              // the wave's rows
        const bool here = first < rows;
        const int32_t tf = (int32_t)(first / a.group), tl = (int32_t)min(it.n - 1, (first + 31) / a.group);
        const int32_t all_lo = win ? it.p0 + tl + 1 - win : 0, all_hi = a.causal ? min(it.cap, it.p0 + tf + 1) : it.cap;
        const int32_t any_lo = win ? it.p0 + tf + 1 - win : 0, any_hi = a.causal ? min(it.cap, it.p0 + tl + 1) : it.cap;

        // ---- queries: column l32, elements 16 s + 8 half ..
        v8 qf[NS][DK / 16];
        float c = a.scale == 0.f ? 1.f : a.scale * 1.4426950408889634f;   // scale * log2(e), by row
        {
            const bool real = row < rows && a.scale != 0.f;           // scale 0: every score is 0
            const AT * q = (const AT *)a.q + (it.r0 + tok) * a.q_tok + head * a.q_head + 8 * half;
            Eight<AT> x[DK / 16];
            float top = 0.f;
#pragma unroll
            for (int s = 0; s < DK / 16; ++s) {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[s].v[j] = (AT)0.f;
                if (real && 16 * s + 8 * half < a.dk) x[s] = load8(q + 16 * s);
            }
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
        const uint64_t zero = (uint64_t)(uintptr_t)g_attn_zero;
        const uint32_t * tab = a.table + (uint64_t)it.seq * a.table_stride;
        auto issue_tab = [&](uint32_t t) {                            // page numbers of tile t: lane l's key
            const int32_t key = key0 + (int32_t)(t * KT + lane);
            const uint32_t pg = (uint32_t)min(key, max(it.cap - 1, 0)) >> a.sh;
            dma4(it.cap > 0 ? (uint64_t)(uintptr_t)(tab + pg) : zero, tab_at + (t & 1) * 256);
        };
        // this wave's part of tile t's rows; returns the keys that a row of the strip
        // sees and that have a page, a bit each
        auto issue_kv = [&](uint32_t t, uint32_t stage) -> uint64_t {
            const int32_t k0 = key0 + (int32_t)(t * KT);
            const uint32_t * pgs = (const uint32_t *)(tabs + (t & 1) * 256);
            const uint32_t own = pgs[lane];
            const int32_t key = k0 + (int32_t)lane;
            const uint64_t vm = __ballot(key >= it.lo && key < it.hi && own < a.n_pages);
            const bool in = (vm >> lane) & 1;
            const uint32_t at = sm_at + stage * P::STAGE, ln = fresh(lane), tok = (uint32_t)key & a.pmask, rows_at = tab_at + 512;
            uint64_t * rows_of = (uint64_t *)(tabs + 512);
            rows_of[lane] = in ? row_at(kb, own, a.k_page, tok, a.k_tok) : zero;
            rows_of[64 + lane] = in ? row_at(vb, own, a.v_page, tok, a.v_tok) : zero;
            dma_rows<DK, false, NK>(rows_at, wave * NK, ln, a.dk, zero, at);
            dma_rows<DV, true, NV>(rows_at + 512, wave * NV, ln, a.dv, zero, at + KT * DK * 2);
            return vm;
        };

        float m, l;
        f32x16 o[DB];
        auto tile = [&](int32_t k0, uint64_t vm, uint32_t at) {
            f32x16 s[2];
            const uint32_t ka = fresh(at + k_lane), va[2] = {fresh(at + v_lane[0]), fresh(at + v_lane[1])};
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[b][i] = 0.f;
            // K in steps of 32 elements: a step's four operands are read while the step
            // before is multiplied
            v8 kf[2][2][2];
            auto ld_k = [&](int step) {
#pragma unroll
                for (int d = 0; d < 2; ++d)
#pragma unroll
                    for (int b = 0; b < 2; ++b) kf[step & 1][d][b] = ld_row<T>(piece<DK>(ka, 4 * step + 2 * d) + 32 * b * DK * 2);
            };
            ld_k(0);
#pragma unroll
            for (int step = 0; step < DK / 32; ++step) {
                __builtin_amdgcn_sched_barrier(0);
                if (step + 1 < DK / 32) ld_k(step + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int d = 0; d < 2; ++d)
#pragma unroll
                    for (int t2 = NS - 1; t2 >= 0; --t2)
#pragma unroll
                        for (int b = 0; b < 2; ++b) s[b] = mma32(kf[step & 1][d][b], qf[t2][2 * step + d], s[b]);
            }
            __builtin_amdgcn_sched_barrier(0);
            // V in steps of 16 keys and up to 128 columns, the same way; the first one is
            // read behind the scores
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
            ld_v(0);
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
            float sum = 0.f;
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    s[b][i] = __builtin_amdgcn_exp2f(fmaf(s[b][i], c, -base)) * weight_unit<T>();
                    sum += s[b][i];
                }
            l += sum;
            v8 pf[NS];
#pragma unroll
            for (int step = 0; step < VSTEPS; ++step) {
                const int k = step / (DB / DC), d0 = step % (DB / DC) * DC;
                __builtin_amdgcn_sched_barrier(0);
                if (step + 1 < VSTEPS) ld_v(step + 1);
                __builtin_amdgcn_sched_barrier(0);
                if (d0 == 0)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        T h[NS];
                        split<T, NS>(s[k >> 1][8 * (k & 1) + j], h);
#pragma unroll
                        for (int t2 = 0; t2 < NS; ++t2) pf[t2][j] = h[t2];
                    }
#pragma unroll
                for (int t2 = NS - 1; t2 >= 0; --t2)
#pragma unroll
                    for (int d = 0; d < DC; ++d) o[d0 + d] = mma32(vf[step & 1][d], pf[t2], o[d0 + d]);
            }
        };
        {
            m = -INFINITY;
            l = 0.f;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
            // order of issue: T0, T1 KV0, T2 KV1, ..: a tile's pages are behind the tile before
            uint64_t vm0 = 0, vm1 = 0;
            issue_tab(0);
            issue_tab(1);
            wait_vm<1>();
            vm0 = issue_kv(0, 0);
            if (nt > 1) {
                issue_tab(2);
                wait_vm<ND + 1>();
                vm1 = issue_kv(1, 1);
            }
            uint32_t stage = 0;
            for (uint32_t t = 0; t < nt; ++t) {
                if (t + 1 < nt) wait_vm<ND + 1>();
                else wait_vm<0>();
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");   // all parts of tile t are there
                const uint64_t vm = vm0;
                vm0 = vm1;
                vm1 = 0;
                const int32_t k0 = key0 + (int32_t)(t * KT);
                if (here && vm && k0 < any_hi && k0 + KT > any_lo) tile(k0, vm, sm_at + stage * P::STAGE);
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");   // the stage has been read
                if (t + 2 < nt) {
                    issue_tab(t + 3);
                    wait_vm<ND + 1>();
                    vm1 = issue_kv(t + 2, stage);
                }
                stage ^= 1;
            }
            wait_vm<0>();
            odd = odd || !finite(l);
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) odd = odd || !finite(o[d][i]);
        }
        l += xor_lane(l, 32, lane);
        if (row < rows) {
            if (begins && ends) {
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
        u += nt;
    }
    const uint32_t any = __ballot(odd) != 0;
    if (lane == 0) sm_odd[wave] = any;
    __syncthreads();
    if (threadIdx.x == 0) {
        uint32_t f = 0;
        for (int i = 0; i < W; ++i) f |= sm_odd[i];
        AttnNote * n = attn_notes<M, DV>(a) + w;
        n->odd = f;
        n->wgs = Ge;
    }
}

namespace {
template <typename AT, typename T, int DK, int DV> int go(const AttnArgs & a, hipStream_t s) {
    typedef PreShape<DK, DV> P;
    const void * k = (const void *)k_attn_pre<AT, T, DK, DV>;
    if (int rc = lds_fits(k, P::LDS, "k_attn_pre")) return rc;
    hipLaunchKernelGGL((k_attn_pre<AT, T, DK, DV>), dim3(a.grid), dim3(64 * P::W), P::LDS, s, a);
    if (int rc = hip_check(hipGetLastError(), "k_attn_pre launch")) return rc;
    hipLaunchKernelGGL((k_attn_join<AT, T, P::M, P::KT, DV, 1>), dim3(a.grid, P::M / 16), dim3(256), 0, s, a);
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
template <int DK, int DV> void shape(AttnPlan & p, uint32_t & per_cu) {
    p.dv = DV;
    p.m = PreShape<DK, DV>::M;
    per_cu = (uint32_t)(160 * 1024 / PreShape<DK, DV>::LDS);
}
}  // namespace

AttnPlan attn_pre_plan(const AttnArgs & a) {
    AttnPlan p{};
    uint32_t per_cu = 1;
    switch (attn_dims(a)) {
        case 0: shape<64, 64>(p, per_cu); break;
        case 1: shape<128, 128>(p, per_cu); break;
        case 2: shape<192, 128>(p, per_cu); break;
        default: shape<256, 256>(p, per_cu); break;
    }
    p.grid = (uint32_t)num_cus() * (per_cu < 1 ? 1 : per_cu > 2 ? 2 : per_cu);
    p.min_units = 2;
    p.ws = attn_ws(p.grid, p.m, p.dv);
    return p;
}

int launch_attn_pre(const AttnArgs & a, uint32_t dtype, uint32_t cache_dtype, hipStream_t s) {
    if (dtype == FLH_DT_F32) return cache_dtype == FLH_DT_F16 ? dims<float, _Float16>(a, s) : dims<float, __bf16>(a, s);
    return dtype == FLH_DT_F16 ? dims<_Float16, _Float16>(a, s) : dims<__bf16, __bf16>(a, s);
}

}  // namespace flh
