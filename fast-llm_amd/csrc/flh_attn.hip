// flh_attn.hip -- attention of new tokens over the paged key/value cache: which
// kernel takes a call.
#include "flh_attn.h"
#include "flh_status.h"

namespace flh {

// Up to 32 rows of a request per kv head: the streaming kernel, which has two blocks of
// 16 rows at most.  At 32 rows 4 requests of 131072 keys take 364 us there and 377 in
// the other one, 16 requests in fp32 over bf16 76 and 96 (in f16, 4096 keys a request, 59 and
// 52); at 48 rows, two strips, 611 and 388, 129 and 101 (104 and 56).
static bool few(const AttnTreeArgs & a) { return (uint64_t)a.max_q * a.group <= 32; }
static AttnPlan plan_of(const AttnTreeArgs & a, uint32_t dtype) { return few(a) ? attn_dec_plan(a) : attn_pre_plan(a, dtype); }

size_t attn_ws_bytes(const AttnTreeArgs & a, uint32_t dtype) { return plan_of(a, dtype).ws; }

int launch_attn(const AttnTreeArgs & args, uint32_t dtype, uint32_t cache_dtype, hipStream_t s) {
    AttnTreeArgs a = args;
    const AttnPlan p = plan_of(a, dtype);
    a.grid = p.grid;
    a.min_units = p.min_units;
    return few(a) ? launch_attn_dec(a, dtype, cache_dtype, s) : launch_attn_pre(a, dtype, cache_dtype, s);
}

}  // namespace flh
