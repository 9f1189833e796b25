// Arguments of shared-prefix attention (prefix_attention.hip), filled by the C entry in api_ops.hip after its checks.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace cmdi {

struct PrefixAttnArgs {
    const void *q, *pk, *pv, *ok, *ov;
    int64_t q_bs, q_ss, q_hs;            // elements between samples / tokens / heads
    int64_t pk_ss, pk_hs, pv_ss, pv_hs;
    int64_t ok_bs, ok_ss, ok_hs, ov_bs, ov_ss, ov_hs;
    const int32_t* own_len;              // [batch] on the device, or null: own_max for all
    int32_t batch, queries, heads, kv_heads, dim, prefix, own_max, causal, dtype;
    float scale;
    void* out;                           // [batch, queries, heads, dim]
    float* lse;                          // [batch, heads, queries] or null
    float* work;                         // partial results: prefix_attention_work_floats
};
// How the work is cut (prefix_attention_plan): one or two launches over (row tile, key chunk) items, then a join where a row
// has several partial results.
struct PrefixAttnLaunch {
    int32_t packed;                      // rows of all samples together (prefix keys only)
    int32_t by_wave;                     // at most 32 rows: a wave a key tile;  else tiles of 128 rows, 32 a wave
    int32_t k_begin, k_end;              // range on the axis [prefix keys | own keys]
    int32_t chunk, chunks, tiles, slot0;
};
struct PrefixAttnPlan {
    int32_t n = 0, slots = 0;
    PrefixAttnLaunch l[2];
};
PrefixAttnPlan prefix_attention_plan(const PrefixAttnArgs& a, int cus);
int64_t prefix_attention_work_floats(const PrefixAttnArgs& a, const PrefixAttnPlan& p);
hipError_t launch_prefix_attention(const PrefixAttnArgs& a, const PrefixAttnPlan& p, hipStream_t stream);

}  // namespace cmdi
