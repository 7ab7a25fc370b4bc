// flh_attn.hip -- attention of new tokens over the paged key/value cache: which
// kernel takes a call.
#include "flh_attn.h"
#include "flh_status.h"

namespace flh {

static AttnPlan plan_of(const AttnArgs & a) { return attn_dec_plan(a); }

size_t attn_ws_bytes(const AttnArgs & a, uint32_t, uint32_t) { return plan_of(a).ws; }

int launch_attn(const AttnArgs & args, uint32_t dtype, uint32_t cache_dtype, hipStream_t s) {
    AttnArgs a = args;
    const AttnPlan p = plan_of(a);
    a.grid = p.grid;
    a.min_units = p.min_units;
    return launch_attn_dec(a, dtype, cache_dtype, s);
}

}  // namespace flh
