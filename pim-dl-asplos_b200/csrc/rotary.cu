// Rotary positions with several axes: pair i of a head turns by angle positions[axis(i)] * inv_freq[i],
//   (a, b) -> (a cos - b sin, b cos + a sin),   sin negated for the inverse (the gradient of a rotation)
// A pair is elements (i, i + pairs) of a head or (2i, 2i + 1); axis(i) by sections, the pairs that each axis has in turn.
// Elements behind the pairs are copied.
//
// Bound by memory: every element is read and written once.  A CTA takes a few tokens: its threads first compute their sines and
// cosines, once per token for all heads, then go through the heads, 16 bytes of either half of the pairs a thread.
// Angles are products in 64 bits, in turns: in 32 bits the angle of position 10^6 is off by 0.03.  What is left after whole turns
// are taken off is split into an fp32 number and its rest, so that cos and sin come out to 32 bits.
#include "dense.cuh"
#include "kernels.h"

#include <type_traits>

namespace lutamm {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kTableFloats = 4096;   // sines and cosines of a CTA's tokens

// E pairs at a time: 16 bytes of either half, or (interleaved) 16 bytes of E / 2 pairs twice.
template <typename T, int E, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) rotary_kernel(RotaryArgs a, uint32_t tokens_per_cta) {
    extern __shared__ float2 s_turn[];   // [token][pair]
    const uint64_t all = (uint64_t)a.batch * a.tokens, t0 = (uint64_t)blockIdx.x * tokens_per_cta;
    const uint32_t n = (uint32_t)(all - t0 < tokens_per_cta ? all - t0 : tokens_per_cta);
    for (uint32_t i = threadIdx.x; i < n * a.pairs; i += kThreads) {
        const uint32_t local = i / a.pairs, pair = i - local * a.pairs;
        const uint64_t token = t0 + local;
        const uint32_t b = (uint32_t)(token / a.tokens), tk = (uint32_t)(token - (uint64_t)b * a.tokens);
        const uint32_t axis = (pair >= a.ends[0]) + (pair >= a.ends[1]) + (pair >= a.ends[2]);
        const int32_t pos = __ldg(a.positions + (int64_t)b * a.position_batch_stride + (int64_t)tk * a.position_token_stride + axis);
        double turns = (double)pos * (double)__ldg(a.inv_freq + pair) * 0.15915494309189535;   // 1 / 2 pi
        turns -= rint(turns);
        const float hi = (float)turns, lo = 6.2831853f * (float)(turns - (double)hi);
        float sn, cs;
        sincospif(2.f * hi, &sn, &cs);
        const float c = fmaf(-lo, sn, cs), s = fmaf(lo, cs, sn);
        s_turn[i] = make_float2(c, a.inverse ? -s : s);
    }
    __syncthreads();
    // units: E pairs each, then the elements that are only copied
    const uint32_t turned = a.pairs / E, units = turned + (a.head_dim - 2 * a.pairs) / E, per_token = units * a.heads;
    for (uint32_t i = threadIdx.x; i < n * per_token; i += kThreads) {
        const uint32_t local = i / per_token, rest = i - local * per_token, head = rest / units, u = rest - head * units;
        const uint64_t token = t0 + local;
        const int64_t b = (int64_t)(token / a.tokens), tk = (int64_t)(token - (uint64_t)b * a.tokens);
        const T* x = static_cast<const T*>(a.x) + b * a.x_batch + tk * a.x_token + (int64_t)head * a.x_head;
        T* y = static_cast<T*>(a.out) + b * a.out_batch + tk * a.out_token + (int64_t)head * a.out_head;
        if (u >= turned) {
            if (a.in_place) continue;
            float v[E];
            const uint32_t c = 2 * a.pairs + (u - turned) * E;
            load_elems<T, E>(x + c, v);
            store_elems<T, E>(y + c, v);
            continue;
        }
        const float2* turn = s_turn + local * a.pairs + u * E;
        float p[E], q[E], o[E], r[E];
        const uint32_t c0 = INTERLEAVED ? 2 * u * E : u * E, c1 = c0 + (INTERLEAVED ? E : a.pairs);
        load_elems<T, E>(x + c0, p);
        load_elems<T, E>(x + c1, q);
        if constexpr (INTERLEAVED && E > 1) {
#pragma unroll
            for (int k = 0; k < E / 2; ++k) {
                const float2 f = turn[k], g = turn[E / 2 + k];
                o[2 * k] = p[2 * k] * f.x - p[2 * k + 1] * f.y;
                o[2 * k + 1] = p[2 * k + 1] * f.x + p[2 * k] * f.y;
                r[2 * k] = q[2 * k] * g.x - q[2 * k + 1] * g.y;
                r[2 * k + 1] = q[2 * k + 1] * g.x + q[2 * k] * g.y;
            }
        } else {
#pragma unroll
            for (int k = 0; k < E; ++k) {
                const float2 f = turn[k];
                o[k] = p[k] * f.x - q[k] * f.y;
                r[k] = q[k] * f.x + p[k] * f.y;
            }
        }
        store_elems<T, E>(y + c0, o);
        store_elems<T, E>(y + c1, r);
    }
}

template <typename T>
cudaError_t run_rotary(const RotaryArgs& a, int sm_count, cudaStream_t s) {
    constexpr int E = kPer16<T>;
    const bool vec = a.vec && a.pairs % E == 0 && a.head_dim % E == 0;
    // Tokens of a CTA: as many as the table holds, at most 16, fewer where that leaves SMs without work.
    const uint64_t all = (uint64_t)a.batch * a.tokens;
    uint64_t per = kTableFloats / 2 / (a.pairs ? a.pairs : 1);
    if (per > 16) per = 16;
    const uint64_t even_out = (all + 2 * (uint64_t)sm_count - 1) / (2 * (uint64_t)sm_count);
    if (per > even_out) per = even_out;
    if (per < 1) per = 1;
    const uint64_t ctas = (all + per - 1) / per;
    if (ctas > 0x7FFFFFFFu) return cudaErrorInvalidValue;
    const size_t bytes = (size_t)per * a.pairs * sizeof(float2);   // at most 16 KB: pairs go up to 2048
    auto go = [&](auto kernel) {
        kernel<<<(uint32_t)ctas, kThreads, bytes, s>>>(a, (uint32_t)per);
        return cudaGetLastError();
    };
    if (vec) return a.interleaved ? go(rotary_kernel<T, E, true>) : go(rotary_kernel<T, E, false>);
    return a.interleaved ? go(rotary_kernel<T, 1, true>) : go(rotary_kernel<T, 1, false>);
}

}  // namespace

cudaError_t launch_rotary(const RotaryArgs& a, uint32_t dtype, int sm_count, cudaStream_t s) {
    if (!a.batch || !a.tokens || !a.heads) return cudaSuccess;
    return dtype == 0 ? run_rotary<float>(a, sm_count, s) : dtype == 1 ? run_rotary<__half>(a, sm_count, s) : run_rotary<__nv_bfloat16>(a, sm_count, s);
}

}  // namespace lutamm
