// flh_attn_dec.hip -- attention of few rows per kv head (single tokens, short
// verify steps): the keys and values of a request are read once, so HBM is
// what bounds it.  32 / 8 heads of 128: 4 requests of 131072 keys in bf16 take 358 us
// (6.0 TB/s; a kernel that only reads 4 GiB reaches 6.1, one of 1 GiB 5.7), 64 requests of up to 8192
// keys with fp32 activations over f16 203 us (5.05 TB/s; 188 with equal lengths, 5.7 TB/s), one
// request of 4001 keys 15 us: two launches, each with a chain of loads (lengths, page
// numbers, keys).  16 requests of up to 8 tokens in fp32 over bf16, 73 us: there the products
// of three terms and the splitting bound it.
#include "flh_attn.h"
#include "flh_status.h"

namespace flh {

// A wave streams 32 keys at a time: their rows of K and V come into its own ring
// of LDS stages by DMA (no barrier anywhere in the loop; page numbers come the
// same way, a tile ahead), scores are K Q^T on the matrix cores, so that a
// lane holds one row's scores of 8 keys, which are, as they are, the operand of
// O^T += V^T P^T; V^T comes out of LDS by transposing reads.  The W waves of
// a workgroup take turns of 32 keys of a tile and join their sums at its end.
// Weights go into the products with V in two terms (three in fp32 over bf16) with 16-bit
// activations too: one would cost as much precision as the rounding of the result (4
// requests of 131072 keys in bf16: off by 0.0023 of the results, 0.0016 so, which is that rounding),
// and a second product costs 0 to 2.5% here (358 and 360 us; 64 requests of up to 8192 keys 195 and 198).
template <int DK, int DV> struct DecShape {
    static constexpr int W = DK + DV <= 256 ? 4 : 2;                  // waves
    static constexpr int KT = 32 * W;                                 // keys of a unit
    static constexpr int NST = DK + DV == 320 ? 3 : 2;                // stages
    static constexpr int STAGE = 32 * (DK + DV) * 2;
    static constexpr int TAB = 2 * 256 + 512;                         // page numbers of two tiles (a DMA writes 64), row addresses of one
    static constexpr int WAVE = NST * STAGE + TAB;
    static constexpr int WALK = 6 * 256;                              // AttnWalk::Chunk
    static constexpr size_t LDS = (size_t)W * (WAVE + WALK) + 1088;            // and maxima, sums, flags
};
template <int DK, int DV> constexpr int dec_threads = 64 * DecShape<DK, DV>::W;

template <typename AT, typename T, int DK, int DV, int MT>
__global__ __launch_bounds__((dec_threads<DK, DV>)) void k_attn_dec(AttnArgs a) {
    typedef DecShape<DK, DV> P;
    typedef typename VecOf<T>::v8 v8;
    constexpr int W = P::W, KT = P::KT, NST = P::NST, M = 16 * MT, NS = split_terms<AT, T>(), NW = NS > 1 ? NS : 2;
    constexpr int NK = DK / 16, NV = DV / 16, ND = NK + NV;           // DMAs of a tile
    extern __shared__ __attribute__((aligned(16))) uint8_t sm[];
    const uint32_t lane = threadIdx.x & 63, l16 = lane & 15, q4 = lane >> 4;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    uint8_t * mine = sm + wave * P::WAVE;
    const uint32_t mine_at = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds_at(mine)), tab_at = mine_at + NST * P::STAGE;
    float * sm_m = (float *)(sm + W * P::WAVE), * sm_l = sm_m + W * M;   // [W][M] each
    uint32_t * sm_odd = (uint32_t *)(sm_l + W * M);                      // [W]
    static_assert((2 * W * M + W) * 4 <= 1088, "shared tail");
    static_assert((size_t)M * DV * 4 <= (size_t)NST * P::STAGE, "a wave's sums lie in its stages");

    // the lane's addresses in a stage: K rows l16 (+ 16 kt), pieces q4 (+ 4 d); V
    // rows 4 q4 + l16 / 4 (+ 16 kt), pieces of 16 columns (+ 2 d)
    const uint32_t k_lane = l16 * (DK * 2) + (q4 ^ swz_k<DK>(l16)) * 16;
    const uint32_t v_row = 4 * q4 + (l16 >> 2);
    const uint32_t v_lane = 32 * DK * 2 + v_row * (DV * 2) + (((l16 >> 1) & 1) ^ swz_v<DV>(v_row)) * 16 + (l16 & 1) * 8;
    typedef typename AttnWalk<M, KT, 0>::Chunk Chunk;
    static_assert(sizeof(Chunk) == P::WALK, "chunk");
    AttnWalk<M, KT, 0> walk(a, *(Chunk *)(sm + W * P::WAVE + 1088 + wave * P::WALK));
    const uint32_t U = walk.total(), Ge = attn_wgs(U, a.grid, a.min_units), w = blockIdx.x;
    if (w >= Ge) return;
    uint32_t u = attn_border(w, U, Ge);
    const uint32_t first_u = u;
    const uint32_t end = attn_border(w + 1, U, Ge);
    bool odd = false;                                                 // a sum is not finite, or a row lost its weight
    while (u < end) {
        AttnItem it;
        walk.find(u, it);
        const uint32_t skip = u - it.u0, nt = min(it.tiles - skip, end - u);
        const int32_t key0 = (int32_t)((it.lo / KT + skip) * KT + 32 * wave);   // this wave's first key
        const bool begins = skip == 0, ends = skip + nt == it.tiles;
        if (u == first_u && wave == 0) attn_note<M, DV, 0>(a, w, U, Ge, it, skip);
        const uint32_t rows = it.n * a.group;

        const uint64_t zero = (uint64_t)(uintptr_t)g_attn_zero;
        const uint32_t * tab = a.table + (uint64_t)it.seq * a.table_stride;
        // page numbers of this wave's keys of tile t: one DMA, lane l's key (lanes from 32 on repeat)
        auto issue_tab = [&](uint32_t t) {
            const int32_t key = key0 + (int32_t)(t * KT + (lane & 31));
            const uint32_t pg = (uint32_t)min(key, max(it.cap - 1, 0)) >> a.sh;
            dma4(it.cap > 0 ? (uint64_t)(uintptr_t)(tab + pg) : zero, tab_at + (t & 1) * 256);
        };
        issue_tab(0);                                                 // (they arrive with the queries)

        // ---- the strip's queries, as the second operand: column l16, elements 32 s + 8 q4 ..
        v8 qf[NS][MT][DK / 32];
        float c[MT];                                                  // scale * log2(e), by column
        int32_t rhi[MT], rlo[MT];                                     // keys that the column's row sees
        const int32_t tf = (int32_t)(it.strip * M / a.group), tl = (int32_t)min(it.n - 1, (it.strip * M + M - 1) / a.group);
        const int32_t all_lo = a.window ? it.p0 + tl + 1 - (int32_t)min(a.window, 1u << 30) : 0;
        const int32_t all_hi = a.causal ? min(it.cap, it.p0 + tf + 1) : it.cap;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const uint32_t r = it.strip * M + 16 * mt + l16, tok = r / a.group, head = it.kvh * a.group + r % a.group;
            // scale 0: every score is 0.  A lane with no row or elements behind d reads the
            // first of the item instead.
            const bool real = r < rows && a.scale != 0.f;
            const AT * q = (const AT *)a.q + (it.r0 + (r < rows ? tok : 0u)) * a.q_tok + (r < rows ? head : it.kvh * a.group) * a.q_head;
            rhi[mt] = key_hi(a, it, tok);
            rlo[mt] = key_lo(a, it, tok);
            c[mt] = a.scale == 0.f ? 1.f : a.scale * 1.4426950408889634f;
            Eight<AT> x[DK / 32];
#pragma unroll
            for (int s = 0; s < DK / 32; ++s) {
                const uint32_t e = 32 * s + 8 * q4;
                x[s] = load8(q + (e < a.dk ? e : 0u));
            }
#pragma unroll
            for (int s = 0; s < DK / 32; ++s) x[s].keep(real & (32 * s + 8 * q4 < a.dk));
            int ex = 0;
            if constexpr (NS == 2) {
                // f16 terms: the row's largest element to [2^13, 2^14), and back in c
                float top = 0.f;
#pragma unroll
                for (int s = 0; s < DK / 32; ++s)
#pragma unroll
                    for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf((float)x[s].v[j]));
                top = fmaxf(top, xor_lane(top, 16, lane));
                top = fmaxf(top, xor_lane(top, 32, lane));
                ex = top > 0.f && finite(top) ? 13 - ilogbf(top) : 0;
                c[mt] = fmaxf(ldexpf(c[mt], -ex), 0x1p-126f);         // (c * -inf below)
            }
#pragma unroll
            for (int s = 0; s < DK / 32; ++s)
                if constexpr (NS == 1) {
                    qf[0][mt][s] = __builtin_bit_cast(v8, x[s]);
                    arrived(qf[0][mt][s]);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        T o[NS];
                        split<T, NS>(NS == 2 ? ldexpf(x[s].v[j], ex) : (float)x[s].v[j], o);
#pragma unroll
                        for (int t = 0; t < NS; ++t) qf[t][mt][s][j] = o[t];
                    }
                }
        }

        const uint64_t kb = (uint64_t)(uintptr_t)a.k + it.kvh * a.k_head, vb = (uint64_t)(uintptr_t)a.v + it.kvh * a.v_head;
        // keys that a row of the strip sees and that have a page: bit per key
        auto issue_kv = [&](uint32_t t, uint32_t stage) -> uint32_t {
            const int32_t k0 = key0 + (int32_t)(t * KT);
            const uint32_t * pgs = (const uint32_t *)(mine + NST * P::STAGE + (t & 1) * 256);
            const uint32_t own = pgs[lane & 31];
            const int32_t key = k0 + (int32_t)(lane & 31);
            const bool in = (key >= it.lo) & (key < it.hi) & (own < a.n_pages);
            const uint32_t vm = (uint32_t)__ballot(in);
            const uint32_t at = mine_at + stage * P::STAGE, ln = fresh(lane), tok = (uint32_t)key & a.pmask, rows_at = tab_at + 512;
            uint64_t * rows_of = (uint64_t *)(mine + NST * P::STAGE + 512);   // K rows, V rows
            const bool isk = lane < 32;
            const uint64_t from = fresh(row_at(isk ? kb : vb, own, isk ? a.k_page : a.v_page, tok, isk ? a.k_tok : a.v_tok));
            rows_of[lane] = in ? from : zero;
            dma_rows<DK, false, NK>(rows_at, ln, a.dk, zero, at);
            dma_rows<DV, true, NV>(rows_at + 256, ln, a.dv, zero, at + 32 * DK * 2);
            return vm;
        };

        float m[MT], l[MT];
        f32x4 o[MT][DV / 16];
        auto tile = [&](int32_t k0, uint32_t vm, uint32_t at) {
            f32x4 s[MT][2];
            const uint32_t ka = fresh(at + k_lane), va = fresh(at + v_lane);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) s[mt][0] = s[mt][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int d = 0; d < DK / 32; ++d)
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) {
                    const v8 kf = ld_row<T>(piece<DK>(ka, 4 * d) + 16 * kt * DK * 2);
#pragma unroll
                    for (int t2 = NS - 1; t2 >= 0; --t2)
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) s[mt][kt] = mma16(kf, qf[t2][mt][d], s[mt][kt]);
                }
            const bool whole = vm == 0xFFFFFFFFu && k0 >= all_lo && k0 + 32 <= all_hi;
            v8 pf[NW][MT];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                float x[8], top = -INFINITY;
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = s[mt][j >> 2][j & 3];
                if (!whole) {
                    const uint32_t see = fresh((vm & (uint32_t)bits_of(rlo[mt] - k0, rhi[mt] - k0)) >> (4 * q4));
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = seen(x[j], see, 16 * (j >> 2) + (j & 3));
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) top = fmaxf(top, x[j]);
                top = fmaxf(top, xor_lane(top, 16, lane));
                top = fmaxf(top, xor_lane(top, 32, lane));
                top *= c[mt];
                if (__ballot(top > m[mt] + MAX_SLACK)) {
                    const float mn = top > m[mt] + MAX_SLACK ? top : m[mt], al = fresh(mn == m[mt] ? 1.f : __builtin_amdgcn_exp2f(m[mt] - mn));
                    m[mt] = mn;
                    l[mt] *= al;
#pragma unroll
                    for (int d = 0; d < DV / 16; ++d) o[mt][d] *= al;
                }
                const float base = m[mt] == -INFINITY ? 0.f : m[mt];
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float p = __builtin_amdgcn_exp2f(fmaf(x[j], c[mt], -base)) * weight_unit<T>();
                    sum += p;
                    T h[NW];
                    split<T, NW>(p, h);
#pragma unroll
                    for (int t2 = 0; t2 < NW; ++t2) pf[t2][mt][j] = h[t2];
                }
                l[mt] += sum;
            }
#pragma unroll
            for (int d = 0; d < DV / 16; ++d) {
                v8 vf;
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) {
                    const typename VecOf<T>::v4 r4 = ld_tr<T>(piece<DV>(va, 2 * d) + 16 * kt * DV * 2);
#pragma unroll
                    for (int j = 0; j < 4; ++j) vf[4 * kt + j] = r4[j];
                }
#pragma unroll
                for (int t2 = NW - 1; t2 >= 0; --t2)
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) o[mt][d] = mma16(vf, pf[t2][mt], o[mt][d]);
            }
        };
        {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                m[mt] = -INFINITY;
                l[mt] = 0.f;
#pragma unroll
                for (int d = 0; d < DV / 16; ++d) o[mt][d] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
            // order of issue: T0, T1 KV0, T2 KV1, ..: a tile's pages are behind the tile before
            uint32_t vms[NST];
#pragma unroll
            for (int i = 0; i < NST; ++i) {
                vms[i] = 0;
                if ((uint32_t)i < nt) {
                    issue_tab(i + 1);
                    if (i == 0) wait_vm<1>();
                    else wait_vm<ND + 1>();
                    vms[i] = issue_kv(i, i);
                }
            }
            uint32_t stage = 0;
            for (uint32_t t = 0; t < nt; ++t) {
                const uint32_t left = nt - 1 - t;                     // tiles behind this one
                if (left >= NST - 1) wait_vm<(NST - 1) * (ND + 1)>();
                else if (left == 1) wait_vm<ND + 1>();                // (NST is 2 or 3)
                else wait_vm<0>();
                const uint32_t vm = vms[0];
                if (vm) {
                    const int32_t k0 = key0 + (int32_t)(t * KT);
                    tile(k0, vm, mine_at + stage * P::STAGE);
                }
#pragma unroll
                for (int i = 0; i + 1 < NST; ++i) vms[i] = vms[i + 1];
                vms[NST - 1] = 0;
                if (t + NST < nt) {
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the stage has been read
                    issue_tab(t + NST + 1);
                    wait_vm<ND + 1>();
                    vms[NST - 1] = issue_kv(t + NST, stage);
                }
                stage = stage + 1 == NST ? 0 : stage + 1;
            }
            wait_vm<0>();

            // ---- the waves' sums: to the workgroup's maximum, then added in wave order
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                l[mt] += xor_lane(l[mt], 16, lane);
                l[mt] += xor_lane(l[mt], 32, lane);
                odd = odd || !finite(l[mt]);
#pragma unroll
                for (int d = 0; d < DV / 16; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i) odd = odd || !finite(o[mt][d][i]);
                sm_m[wave * M + 16 * mt + l16] = m[mt];               // (q4: the same value)
            }
            __syncthreads();
        }
        float * so = (float *)mine;                                   // [M][DV]
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const uint32_t r = 16 * mt + l16;
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < W; ++i) top = fmaxf(top, sm_m[i * M + r]);
            const float f = m[mt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[mt] - top);
            sm_l[wave * M + r] = l[mt] * f;
#pragma unroll
            for (int d = 0; d < DV / 16; ++d) {
                f32x4 v = o[mt][d];
                if (m[mt] != -INFINITY) v *= f;
                *(f32x4 *)(so + r * DV + 16 * d + 4 * q4) = v;
            }
        }
        __syncthreads();
        float * part = begins && ends ? nullptr : attn_part<M, DV>(a, w, begins);
        bool lost = false;                                            // a row that has keys got no weight
        for (uint32_t e = threadIdx.x; e < M * DV / 4; e += 64 * W) {
            const uint32_t r = e / (DV / 4), d = e % (DV / 4) * 4, row = it.strip * M + r;
            if (row >= rows) continue;
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < W; ++i) {
                v += *(const f32x4 *)((const float *)(sm + i * P::WAVE) + r * DV + d);
                sum += sm_l[i * M + r];
            }
            if (part) {
                *(f32x4 *)(part + r * DV + d) = v;
                if (d == 0) {
                    float top = -INFINITY;
#pragma unroll
                    for (int i = 0; i < W; ++i) top = fmaxf(top, sm_m[i * M + r]);
                    part[M * DV + r] = top;
                    part[M * (DV + 1) + r] = sum;
                }
            } else if (d < a.dv) {
                const uint32_t tok = it.r0 + row / a.group, head = it.kvh * a.group + row % a.group;
                if (!(sum > 0.f)) lost = lost || key_hi(a, it, row / a.group) > max(key_lo(a, it, row / a.group), 0);
                if (sum == 0.f) v = f32x4{0.f, 0.f, 0.f, 0.f};
                else v /= sum;
                store4((AT *)a.out + tok * a.o_tok + head * a.o_head + d, v[0], v[1], v[2], v[3]);
            }
        }
        if (__ballot(lost)) odd = odd || any_page(a, it, it.lo, it.hi);
        u += nt;
        __syncthreads();                                              // the next item's stages
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
template <typename AT, typename T, int DK, int DV, int MT> int go(const AttnArgs & a, hipStream_t s) {
    typedef DecShape<DK, DV> P;
    constexpr int M = 16 * MT;
    const void * k = (const void *)k_attn_dec<AT, T, DK, DV, MT>;
    if (int rc = lds_fits(k, P::LDS, "k_attn_dec")) return rc;
    hipLaunchKernelGGL((k_attn_dec<AT, T, DK, DV, MT>), dim3(a.grid), dim3(64 * P::W), P::LDS, s, a);
    if (int rc = hip_check(hipGetLastError(), "k_attn_dec launch")) return rc;
    hipLaunchKernelGGL((k_attn_join<AT, T, M, P::KT, DV, 4, 0>), dim3(a.grid, M / 4), dim3(256), 0, s, a);
    return hip_check(hipGetLastError(), "k_attn_join launch");
}
template <typename AT, typename T, int MT> int dims(const AttnArgs & a, hipStream_t s) {
    switch (attn_dims(a)) {
        case 0: return go<AT, T, 64, 64, MT>(a, s);
        case 1: return go<AT, T, 128, 128, MT>(a, s);
        case 2: return go<AT, T, 192, 128, MT>(a, s);
        default: return go<AT, T, 256, 256, MT>(a, s);
    }
}
template <typename AT, typename T> int tiles(const AttnArgs & a, hipStream_t s) {
    return attn_dec_plan(a).m == 16 ? dims<AT, T, 1>(a, s) : dims<AT, T, 2>(a, s);
}
template <int DK, int DV> void shape(AttnPlan & p, uint32_t & per_cu) {
    p.dv = DV;
    per_cu = (uint32_t)(160 * 1024 / DecShape<DK, DV>::LDS);
}
}  // namespace

AttnPlan attn_dec_plan(const AttnArgs & a) {
    AttnPlan p{};
    uint32_t per_cu = 1;
    switch (attn_dims(a)) {
        case 0: shape<64, 64>(p, per_cu); break;
        case 1: shape<128, 128>(p, per_cu); break;
        case 2: shape<192, 128>(p, per_cu); break;
        default: shape<256, 256>(p, per_cu); break;
    }
    p.m = (uint64_t)a.max_q * a.group <= 16 ? 16 : 32;
    p.grid = (uint32_t)num_cus() * (per_cu ? per_cu : 1);
    p.min_units = 1;
    p.ws = attn_ws(p.grid, p.m, p.dv);
    return p;
}

int launch_attn_dec(const AttnArgs & a, uint32_t dtype, uint32_t cache_dtype, hipStream_t s) {
    if (dtype == FLH_DT_F32) return cache_dtype == FLH_DT_F16 ? tiles<float, _Float16>(a, s) : tiles<float, __bf16>(a, s);
    return dtype == FLH_DT_F16 ? tiles<_Float16, _Float16>(a, s) : tiles<__bf16, __bf16>(a, s);
}

}  // namespace flh
