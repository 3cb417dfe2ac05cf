// attn_plan_check.hip -- how a batch's attention is launched (kv_attn_plan.h), for
// the CPU tests: it launches nothing.  Built by inferno_hip.build into
// tests/native/_build/libsdig_check.so.
#include "kv_attn_plan.h"

// rows of a tile, tiles, parts, keys of a part at least, halves, bytes
extern "C" void attn_plan_of(int act, int kv_type, int q_heads, int kv_heads, int dim, int sequences, int tokens,
                             long long capacity, int window, long long *out)
{
    const ihip::AttnPlan p = ihip::attn_plan(act, kv_type, q_heads, kv_heads, dim, sequences, tokens, capacity, window);
    out[0] = p.rows;
    out[1] = p.tiles;
    out[2] = p.splits;
    out[3] = p.least;
    out[4] = p.halves;
    out[5] = (long long)p.bytes;
}
