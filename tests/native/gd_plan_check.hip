// gd_plan_check.hip -- how calls of the gated delta rule and of sampling are laid out
// (gd_plan.h, sample_plan.h), for the CPU tests: it launches nothing.  Built by
// inferno_hip.build into tests/native/_build/libsdig_check.so.
#include "gd_plan.h"
#include "sample_plan.h"

// chunks, steps, numbers of chunks, bytes of K, offsets of P and M, factors, outputs, bytes
extern "C" void delta_plan_of(int parts, int k_heads, int v_heads, int k_dim, int v_dim, long long tokens, long long sequences,
                              int most, long long *out)
{
    const ihip::DeltaPlan p = ihip::delta_plan(parts, k_heads, v_heads, k_dim, v_dim, tokens, sequences, most);
    const long long v[] = {p.chunks, p.steps, p.tiles, p.frag, (long long)p.tri, (long long)p.rows, (long long)p.raw,
                           (long long)p.bytes};
    for (int i = 0; i < 8; ++i)
        out[i] = v[i];
}

extern "C" void sample_plan_of(int rows, int vocab, long long *out)
{
    const ihip::SamplePlan p = ihip::sample_plan(rows, vocab);
    const long long v[] = {p.per, p.slices, p.rows, (long long)p.bounds, (long long)p.bins, (long long)p.merged,
                           (long long)p.list, (long long)p.bytes};
    for (int i = 0; i < 8; ++i)
        out[i] = v[i];
}
