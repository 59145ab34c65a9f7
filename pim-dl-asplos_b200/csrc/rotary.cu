// Rotary positions with several axes: pair i of a head turns by angle positions[axis(i)] * inv_freq[i],
//   (a, b) -> (a cos - b sin, b cos + a sin),   sin negated for the inverse (the gradient of a rotation)
// A pair is elements (i, i + pairs) of a head or (2i, 2i + 1); axis(i) by sections, the pairs that each axis has in turn.
// Elements behind the pairs are copied.
//
// Bound by memory: every element is read and written once.  A CTA takes a few tokens: its threads first compute their sines and
// cosines, once per token for all heads, then go through the heads, 16 bytes of either half of the pairs a thread.
// 12608 tokens, 24 heads of 64 in fp32: 26.3 us, 5.9 TB/s.  16384 tokens, 16 heads of 128 in bf16: 27.4 us, 4.9 TB/s; half the bytes come with each sine, and
// the sines' part of a CTA's time is what three CTAs on an SM hide only in part (loads that leave after them: 28.8).
// Angles are products in 64 bits, in turns: in 32 bits the angle of position 10^6 is off by 0.03.  What is left after whole turns
// are taken off is split into an fp32 number and its rest, so that cos and sin come out to 32 bits.
#include "dense.cuh"
#include "kernels.h"

#include <algorithm>
#include <type_traits>

namespace lutamm {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kTable = 2048;   // sines and cosines of a CTA's tokens: 16 KB

// E pairs at a time: 16 bytes of either half, or (interleaved) 16 bytes of E / 2 pairs twice.
template <typename T, int E, bool INTERLEAVED>
__device__ __forceinline__ void turn_unit(const float (&p)[E], const float (&q)[E], const float2* turn, float (&o)[E], float (&r)[E]) {
    // (one multiplication and one fused one, whichever instance: equal calls on other strides give equal bits)
    auto turned = [](float x, float y, float2 f, float& u, float& v) {
        u = fmaf(x, f.x, -__fmul_rn(y, f.y));
        v = fmaf(y, f.x, __fmul_rn(x, f.y));
    };
    if constexpr (INTERLEAVED && E > 1) {
#pragma unroll
        for (int k = 0; k < E / 2; ++k) {
            turned(p[2 * k], p[2 * k + 1], turn[k], o[2 * k], o[2 * k + 1]);
            turned(q[2 * k], q[2 * k + 1], turn[E / 2 + k], r[2 * k], r[2 * k + 1]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < E; ++k) turned(p[k], q[k], turn[k], o[k], r[k]);
    }
}

// A CTA: `per` tokens of one sequence.
template <typename T, int E, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) rotary_kernel(RotaryArgs a, uint32_t per, uint32_t blocks) {
    extern __shared__ float2 s_turn[];   // [token][pair]
    const uint32_t b = blockIdx.x / blocks, t0 = (blockIdx.x - b * blocks) * per, n = min(per, a.tokens - t0);
    // A unit is E pairs.  A thread has one unit of one token, takes its sines and cosines into registers, and goes through the heads, some on their way.
    const uint32_t units = a.pairs / E, slots = n * units, width = min(max(slots, 1u), (uint32_t)kThreads), groups = kThreads / width, group = threadIdx.x / width;
    const uint32_t slot0 = group < groups ? threadIdx.x - group * width : slots;
    const T* xb = static_cast<const T*>(a.x) + (int64_t)b * a.x_batch + (int64_t)t0 * a.x_token;
    T* yb = static_cast<T*>(a.out) + (int64_t)b * a.out_batch + (int64_t)t0 * a.out_token;
    constexpr int kInFlight = 4;
    Piece<T, E> p_raw[kInFlight], q_raw[kInFlight];
    auto fetch = [&](uint32_t slot, uint32_t first) {
        const uint32_t local = slot / units, u = slot - local * units, c0 = INTERLEAVED ? 2 * u * E : u * E, c1 = c0 + (INTERLEAVED ? E : a.pairs);
        const T* x = xb + (int64_t)local * a.x_token;
#pragma unroll
        for (int k = 0; k < kInFlight; ++k) {
            const uint32_t head = first + k * groups;
            if (head < a.heads) {
                p_raw[k].load(x + (int64_t)head * a.x_head + c0);
                q_raw[k].load(x + (int64_t)head * a.x_head + c1);
            }
        }
    };
    if (slot0 < slots) fetch(slot0, group);   // the first ones while the sines are formed
    for (uint32_t i = threadIdx.x; i < n * a.pairs; i += kThreads) {
        const uint32_t local = i / a.pairs, pair = i - local * a.pairs;
        const uint32_t axis = (pair >= a.ends[0]) + (pair >= a.ends[1]) + (pair >= a.ends[2]);
        const int32_t pos = __ldg(a.positions + (int64_t)b * a.position_batch_stride + (int64_t)(t0 + local) * a.position_token_stride + axis);
        double turns = (double)pos * (double)__ldg(a.inv_freq + pair) * 0.15915494309189535;   // 1 / 2 pi
        turns -= rint(turns);
        const float hi = (float)turns, lo = 6.2831853f * (float)(turns - (double)hi);
        float sn, cs;
        sincospif(2.f * hi, &sn, &cs);
        const float c = fmaf(-lo, sn, cs), s = fmaf(lo, cs, sn);
        s_turn[i] = make_float2(c, a.inverse ? -s : s);
    }
    __syncthreads();
    for (uint32_t slot = slot0; slot < slots; slot += width) {
        const uint32_t local = slot / units, u = slot - local * units;
        float2 turn[E];
#pragma unroll
        for (int k = 0; k < E; ++k) turn[k] = s_turn[slot * E + k];
        const uint32_t c0 = INTERLEAVED ? 2 * u * E : u * E, c1 = c0 + (INTERLEAVED ? E : a.pairs);
        T* y = yb + (int64_t)local * a.out_token;
        for (uint32_t first = group; first < a.heads; first += kInFlight * groups) {
            if (slot != slot0 || first != group) fetch(slot, first);
#pragma unroll
            for (int k = 0; k < kInFlight; ++k) {
                const uint32_t head = first + k * groups;
                if (head < a.heads) {
                    float p[E], q[E], o[E], r[E];
                    p_raw[k].widen(p);
                    q_raw[k].widen(q);
                    turn_unit<T, E, INTERLEAVED>(p, q, turn, o, r);
                    store_elems<T, E>(y + (int64_t)head * a.out_head + c0, o);
                    store_elems<T, E>(y + (int64_t)head * a.out_head + c1, r);
                }
            }
        }
    }
    const uint32_t rest = (a.head_dim - 2 * a.pairs) / E;   // pieces of a head that are only copied
    if (rest == 0 || a.in_place) return;
    for (uint32_t i = threadIdx.x; i < n * a.heads * rest; i += kThreads) {
        const uint32_t local = i / (a.heads * rest), j = i - local * a.heads * rest, head = j / rest, c = 2 * a.pairs + (j - head * rest) * E;
        float v[E];
        load_elems<T, E>(xb + (int64_t)local * a.x_token + (int64_t)head * a.x_head + c, v);
        store_elems<T, E>(yb + (int64_t)local * a.out_token + (int64_t)head * a.out_head + c, v);
    }
}

template <typename T>
cudaError_t run_rotary(const RotaryArgs& a, int sm_count, cudaStream_t s) {
    constexpr uint32_t E = kPer16<T>;
    const bool vec = a.vec && a.pairs % E == 0 && a.head_dim % E == 0;
    // Tokens of a CTA: so many that their units and a quarter of the heads fill it, fewer where that leaves SMs without work; as the table holds.
    const uint32_t units = std::max(1u, a.pairs / (vec ? E : 1));
    uint64_t per = std::max(1u, kThreads / 4 / units);
    per = std::min<uint64_t>(per, ((uint64_t)a.batch * a.tokens + 4 * (uint64_t)sm_count - 1) / (4 * (uint64_t)sm_count));
    per = std::max<uint64_t>(1, std::min<uint64_t>({per, a.tokens, kTable / std::max(1u, a.pairs)}));
    const uint64_t blocks = (a.tokens + per - 1) / per, ctas = blocks * a.batch;
    if (ctas > 0x7FFFFFFFu) return cudaErrorInvalidValue;
    const size_t bytes = (size_t)per * a.pairs * sizeof(float2);   // at most 16 KB: pairs go up to 2048
    auto go = [&](auto kernel) {
        kernel<<<(uint32_t)ctas, kThreads, bytes, s>>>(a, (uint32_t)per, (uint32_t)blocks);
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
