// flh_attn.hip -- attention of new tokens over the paged key/value cache: which
// kernel takes a call.
#include "flh_attn.h"
#include "flh_status.h"

namespace flh {

// up to 32 rows of a request per kv head: the streaming kernel
static bool few(const AttnArgs & a) { return (uint64_t)a.max_q * a.group <= 32; }
static AttnPlan plan_of(const AttnArgs & a, uint32_t dtype) { return few(a) ? attn_dec_plan(a) : attn_pre_plan(a, dtype); }

size_t attn_ws_bytes(const AttnArgs & a, uint32_t dtype, uint32_t) { return plan_of(a, dtype).ws; }

int launch_attn(const AttnArgs & args, uint32_t dtype, uint32_t cache_dtype, hipStream_t s) {
    AttnArgs a = args;
    const AttnPlan p = plan_of(a, dtype);
    a.grid = p.grid;
    a.min_units = p.min_units;
    return few(a) ? launch_attn_dec(a, dtype, cache_dtype, s) : launch_attn_pre(a, dtype, cache_dtype, s);
}

}  // namespace flh
