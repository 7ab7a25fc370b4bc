// flh_attn.hip -- attention of new tokens over the paged key/value cache.
#include "flh_common.h"
#include "flh_internal.h"
#include "flh_status.h"

namespace flh {

// One wave per (row, head), lane per key, one pass with the running maximum and
// sum of the softmax.
template <typename AT, typename CT>
__global__ __launch_bounds__(64) void k_attn_row(AttnArgs a) {
    __shared__ float pr[64];
    __shared__ uint64_t vat[64];
    const uint32_t lane = threadIdx.x, row = blockIdx.x, head = blockIdx.y;
    // the request of this row
    uint32_t s = 0xFFFFFFFFu, r0 = 0, r1 = 0;
    for (uint32_t b = 0; b < a.n_seq; ++b) {
        const uint32_t x = min(a.q_start[b], a.n_tok), y = min(a.q_start[b + 1], a.n_tok);
        if (row >= x && row < y) { s = b; r0 = x; r1 = y; break; }
    }
    if (s == 0xFFFFFFFFu) return;
    const uint32_t kvh = head / a.group;
    const int64_t kv = a.kv_len[s], cap = min(kv, (int64_t)a.table_stride << a.sh);
    const int64_t p = kv - (r1 - r0) + (row - r0);
    const int64_t hi = a.causal ? min(cap, p + 1) : cap, lo = a.window ? max((int64_t)0, p + 1 - a.window) : 0;
    const AT * q = (const AT *)a.q + row * a.q_tok + head * a.q_head;
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int64_t j0 = lo; j0 < hi; j0 += 64) {
        const int64_t j = j0 + lane;
        float t = -INFINITY;
        uint32_t pg = FLH_KV_NONE;
        if (j < hi) pg = a.table[(uint64_t)s * a.table_stride + (j >> a.sh)];
        const uint64_t off = j & ((1u << a.sh) - 1u);
        if (pg < a.n_pages) {
            const CT * k = (const CT *)a.k + (uint64_t)pg * a.k_page + off * a.k_tok + (uint64_t)kvh * a.k_head;
            t = 0.f;
            for (uint32_t i = 0; i < a.dk; ++i) t = fmaf((float)q[i], (float)k[i], t);
            t *= a.scale;
        }
        float mt = t;
        for (int x = 1; x < 64; x <<= 1) mt = fmaxf(mt, __shfl_xor(mt, x));
        const float mn = fmaxf(m, mt), ms = mn == -INFINITY ? 0.f : mn;
        const float e = expf(t - ms), al = expf(m - ms);
        float sum = e;
        for (int x = 1; x < 64; x <<= 1) sum += __shfl_xor(sum, x);
        l = l * al + sum;
        m = mn;
        pr[lane] = e;
        vat[lane] = pg < a.n_pages ? (uint64_t)pg * a.v_page + off * a.v_tok + (uint64_t)kvh * a.v_head : ~0ull;
        __syncthreads();
        for (uint32_t c = 0; c < 4; ++c) o[c] *= al;
        for (uint32_t k = 0; k < 64; ++k) {
            if (vat[k] == ~0ull) continue;
            for (uint32_t c = 0; c < 4; ++c)
                if (64 * c + lane < a.dv) o[c] = fmaf(pr[k], (float)((const CT *)a.v)[vat[k] + 64 * c + lane], o[c]);
        }
        __syncthreads();
    }
    for (uint32_t c = 0; c < 4; ++c)
        if (64 * c + lane < a.dv)
            ((AT *)a.out)[row * a.o_tok + head * a.o_head + 64 * c + lane] = (AT)(l == 0.f ? 0.f : o[c] / l);
}

size_t attn_ws_bytes(const AttnArgs &, uint32_t, uint32_t) { return 0; }

int launch_attn(const AttnArgs & a, uint32_t dtype, uint32_t cache_dtype, hipStream_t s) {
    const dim3 g(a.n_tok, a.group * a.n_kv);
    if (dtype == FLH_DT_F32 && cache_dtype == FLH_DT_F16) hipLaunchKernelGGL((k_attn_row<float, _Float16>), g, dim3(64), 0, s, a);
    else if (dtype == FLH_DT_F32) hipLaunchKernelGGL((k_attn_row<float, __bf16>), g, dim3(64), 0, s, a);
    else if (dtype == FLH_DT_F16) hipLaunchKernelGGL((k_attn_row<_Float16, _Float16>), g, dim3(64), 0, s, a);
    else hipLaunchKernelGGL((k_attn_row<__bf16, __bf16>), g, dim3(64), 0, s, a);
    return hip_check(hipGetLastError(), "k_attn_row launch");
}

}  // namespace flh
