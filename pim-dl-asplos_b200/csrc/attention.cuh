// What the attention kernels share: which keys a query sees, and access to the other CTAs of a cluster.
//
// Query i of sequence b stands at position p = first[b] + i.  It sees key j if j < lengths[b], j <= p + right and
// (j >= p - left or j < sinks); a negative bound is none.
#pragma once
#include "dense.cuh"
#include "kernels.h"

namespace lutamm {

struct KeyBounds {   // of one query: the keys lo .. hi - 1 and those in front of `sinks` (and of hi)
    int32_t lo, hi;
};
__device__ __forceinline__ int32_t clamp_key(int64_t v, int32_t most) { return v < 0 ? 0 : v > most ? most : (int32_t)v; }
__device__ __forceinline__ KeyBounds key_bounds(const AttentionArgs& a, int64_t position, int32_t length) {
    KeyBounds k;
    k.hi = a.right < 0 ? length : clamp_key(position + a.right + 1, length);
    k.lo = a.left < 0 ? 0 : clamp_key(position - a.left, k.hi);
    return k;
}

// The keys that some query at positions first .. last sees: the sinks 0 .. sinks - 1, then lo .. hi - 1.
struct KeySpan {
    int32_t sinks, lo, hi;
};
__device__ __forceinline__ KeySpan key_span(const AttentionArgs& a, int64_t first, int64_t last, int32_t length) {
    KeySpan s;
    s.hi = key_bounds(a, last, length).hi;
    s.lo = a.left < 0 ? 0 : clamp_key(first - a.left, s.hi);
    s.sinks = (uint32_t)s.lo < a.sinks ? s.lo : (int32_t)a.sinks;
    return s;
}
__device__ __forceinline__ int32_t key_count(const AttentionArgs& a, uint32_t b) {
    if (!a.lengths) return (int32_t)a.keys;
    const int32_t n = __ldg(a.lengths + b);
    return n < 0 ? 0 : n > (int32_t)a.keys ? (int32_t)a.keys : n;
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float load_shared_cluster(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float4 load_shared_cluster4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

}  // namespace lutamm
