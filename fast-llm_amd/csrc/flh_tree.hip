// flh_tree.hip -- trees of drafted tokens: what a row of a tree sees, from its parents.
#include "flh_common.h"
#include "flh_internal.h"
#include "flh_status.h"

namespace flh {

// Thread per row (x) and word of 32 rows (y): it walks up from its row, as far as the
// word's first one (a parent's index is below its child's, so the walk ends).  The requests' first rows
// and the workgroup's parents are read once into LDS, else the search and the walk would be
// chains of loads from memory.  A launch and two rounds of loads bound it: 8 trees of 5 to 16 rows 3.2 us, 300
// of up to 100 rows (15000 in all, 4 words each) 9.5.
constexpr uint32_t TREE_T = 256, TREE_SEQ = 2048, TREE_ROWS = 4096;

__global__ __launch_bounds__(TREE_T) void k_tree_plan(flh_tree_plan_p p) {
    __shared__ uint32_t first[TREE_SEQ];
    __shared__ int32_t up[TREE_ROWS];
    const uint32_t row0 = blockIdx.x * TREE_T, row = row0 + threadIdx.x, end = min(p.q_start[p.n_seq], p.n_tok);
    if (row0 >= end) return;
    const bool lds = p.n_seq <= TREE_SEQ;
    if (lds) {
        for (uint32_t i = threadIdx.x; i < p.n_seq; i += TREE_T) first[i] = p.q_start[i];
        __syncthreads();
    }
    const uint32_t * at = lds ? first : p.q_start;
    // the last request that begins at or before a row (empty ones begin where the next does)
    auto owner = [&](uint32_t r) {
        uint32_t lo = 0, n = p.n_seq;
        while (n > 1) {
            const uint32_t h = n >> 1;
            if (at[lo + h] <= r) { lo += h; n -= h; }
            else n = h;
        }
        return lo;
    };
    // parents of the rows from the first one's request on
    const uint32_t base = at[owner(row0)], have = base <= row0 ? min(end - base, TREE_ROWS) : 0;
    for (uint32_t i = threadIdx.x; i < min(have, row0 + TREE_T - base); i += TREE_T) up[i] = p.parent[base + i];
    __syncthreads();
    if (row >= end) return;
    const uint32_t s = owner(row), r0 = at[s];
    if (r0 > row) return;                                         // in front of the first request
    const uint32_t w = blockIdx.y;
    const int32_t r = (int32_t)(row - r0);
    uint32_t bits = 0, dist = 0;
    for (int32_t x = r;;) {
        if ((uint32_t)x >> 5 == w && (p.window == 0 || dist < p.window)) bits |= 1u << (x & 31);
        const uint32_t i = r0 + (uint32_t)x - base;
        const int32_t next = i < TREE_ROWS && i < have ? up[i] : p.parent[r0 + (uint32_t)x];
        if (next < 0 || next >= x || (w && (uint32_t)next < 32 * w)) break;
        x = next;
        ++dist;
    }
    p.mask[(uint64_t)row * p.mask_stride + w] = bits;
    if (w == 0) {
        p.depth[row] = dist;
        if (p.pos) p.pos[row] = (int32_t)(p.kv_len[s] - (p.q_start[s + 1] - r0) + dist);
    }
}

int launch_tree_plan(const flh_tree_plan_p & p, hipStream_t s) {
    hipLaunchKernelGGL(k_tree_plan, dim3((p.n_tok + TREE_T - 1) / TREE_T, p.mask_stride), dim3(TREE_T), 0, s, p);
    return hip_check(hipGetLastError(), "k_tree_plan launch");
}

}  // namespace flh
