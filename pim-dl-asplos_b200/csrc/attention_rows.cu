// Attention for few rows (query tokens times the query heads that share a key head): single tokens behind a cache.
//   s_j = q k_j scale,  out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m)   over the keys that the query sees (attention.cuh)
//
// Bound by memory for one or two rows, by instructions for eight: keys and values are read once for up to eight rows.  8 x 8192 keys, 16 heads of
// 128, one row: fp32 172 us, 6.2 TB/s, bf16 94 us, 5.7 TB/s; eight rows of fp32 319 us, 3.4 TB/s.  LPK lanes share a key, 16 bytes each; each such group of
// lanes walks keys of its own, four at a time, with a maximum, a sum and an output of its own (the running form of the softmax), so
// nothing is exchanged between groups before the end.  The rows' partial products are summed over the lanes of a group by halves: after
// each exchange a lane holds half as many rows, in the end the score of one.  The keys of one head and sequence are split
// over the CTAs of a cluster where there would be too few CTAs; they join through distributed shared memory: no scratch
// memory, no second launch, one order of summation.
// Scores, maxima, sums and outputs are fp32; weights are not rounded, but all brought down by a power of two no less than the number of keys, so that sums
// of values do not overflow where their mean does not.
#include "attention.cuh"
#include "ptx.cuh"

#include <type_traits>

namespace lutamm {
namespace {

constexpr int kThreads = 128, kWarps = kThreads / 32;
constexpr int kUnroll = 4;
constexpr int kMostHead = 128;

template <typename T, int E>
__device__ __forceinline__ void load_row(const T* p, bool vec, uint32_t c, uint32_t dim, float (&v)[E]) {
    if (vec) {
        if (c < dim) { load_elems<T, E>(p + c, v); return; }
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = 0.f;
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = c + i < dim ? to_float(p[c + i]) : 0.f;
    }
}

template <typename T>
__device__ __forceinline__ uint4 load_16(const T* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }
template <typename T, int E>
__device__ __forceinline__ void widen(const uint4& w, float (&v)[E]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
            v[i] = __uint_as_float(u[i]);
        } else {
            const float2 f = unpack2(u[i], static_cast<T*>(nullptr));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}

// VEC: all tensors start on 16 bytes throughout.
template <typename T, int LPK, int RB, bool VEC>
__global__ void __launch_bounds__(kThreads) attention_rows_kernel(AttentionArgs a, uint32_t row_groups) {
    constexpr int E = kPer16<T>, kGroups = 32 / LPK, kStreams = kWarps * kGroups, kStep = LPK / RB;
    static_assert(RB <= LPK);
    __shared__ float s_m[kWarps + 1][RB], s_l[kWarps + 1][RB];
    __shared__ float s_acc[kWarps][RB][kMostHead];   // [0] becomes the CTA's
    const uint32_t shares = cluster_size_x(), share = cluster_rank();
    uint64_t item = blockIdx.x / shares;
    const uint32_t rg = (uint32_t)(item % row_groups);
    item /= row_groups;
    const uint32_t g = (uint32_t)(item % a.kv_heads), b = (uint32_t)(item / a.kv_heads);
    const uint32_t per_head = a.heads / a.kv_heads;
    const uint64_t rows = (uint64_t)a.queries * per_head, r0 = (uint64_t)rg * RB;
    const uint32_t n_rows = rows - r0 < RB ? (uint32_t)(rows - r0) : RB;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, in_key = lane % LPK, group = lane / LPK;
    const uint32_t c = in_key * E;

    const int32_t length = key_count(a, b);
    const int64_t first = a.first ? __ldg(a.first + b) : 0;
    const int64_t p0 = first + (int64_t)(r0 / per_head), p1 = first + (int64_t)((r0 + n_rows - 1) / per_head);
    const KeySpan span = key_span(a, p0, p1, length);
    const uint32_t n_keys = (uint32_t)(span.sinks + (span.hi - span.lo));
    const float down = __int_as_float((n_keys <= 1 ? 127 : 95 + __clz(n_keys - 1)) << 23);   // 2^-k, 2^k no less than n_keys
    const uint32_t t0 = (uint32_t)((uint64_t)n_keys * share / shares), t1 = (uint32_t)((uint64_t)n_keys * (share + 1) / shares);

    float q[RB][E];
#pragma unroll
    for (int r = 0; r < RB; ++r) {
        if ((uint32_t)r < n_rows) {
            const uint64_t row = r0 + r;
            const uint64_t i = row / per_head;
            const uint32_t h = g * per_head + (uint32_t)(row - i * per_head);
            load_row<T, E>(static_cast<const T*>(a.q) + (int64_t)b * a.q_batch + (int64_t)i * a.q_token + (int64_t)h * a.q_head, VEC, c, a.head_dim, q[r]);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) q[r][e] = 0.f;
        }
    }
    // this lane's row, its bounds
    const uint32_t my_row = in_key / kStep;
    const KeyBounds mine = key_bounds(a, first + (int64_t)((r0 + (my_row < n_rows ? my_row : n_rows - 1)) / per_head), length);
    const T* kp = static_cast<const T*>(a.k) + (int64_t)b * a.k_batch + (int64_t)g * a.k_head;
    const T* vp = static_cast<const T*>(a.v) + (int64_t)b * a.v_batch + (int64_t)g * a.v_head;

    float m = -INFINITY, l = 0.f, acc[RB][E];
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int e = 0; e < E; ++e) acc[r][e] = 0.f;

    const uint32_t stream = warp * kGroups + group;
    // The next four keys and values are on their way while these are worked on, as raw bytes.
    uint4 k_raw[kUnroll], v_raw[kUnroll];
    auto key_at = [&](uint32_t t) -> uint32_t { return t < (uint32_t)span.sinks ? t : (uint32_t)span.lo + (t - (uint32_t)span.sinks); };
    auto fetch = [&](uint32_t base) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const uint32_t t = base + u * kStreams + stream;
            k_raw[u] = v_raw[u] = make_uint4(0, 0, 0, 0);
            if (t < t1 && c < a.head_dim) {
                const int64_t key = key_at(t);
                k_raw[u] = load_16(kp + key * a.k_token + c);
                v_raw[u] = load_16(vp + key * a.v_token + c);
            }
        }
    };
    if (VEC && t0 < t1) fetch(t0);
    for (uint32_t base = t0; base < t1; base += kUnroll * kStreams) {   // (t1 - t0 and this stay below 2^31 + 2^9)
        float kf[kUnroll][E], vf[kUnroll][E], s[kUnroll];
        uint32_t key[kUnroll];
        bool in[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const uint32_t t = base + u * kStreams + stream;
            in[u] = t < t1;
            key[u] = in[u] ? key_at(t) : 0u;
            if constexpr (VEC) {
                widen<T, E>(k_raw[u], kf[u]);
                widen<T, E>(v_raw[u], vf[u]);
            } else if (in[u]) {
                load_row<T, E>(kp + (int64_t)key[u] * a.k_token, false, c, a.head_dim, kf[u]);
                load_row<T, E>(vp + (int64_t)key[u] * a.v_token, false, c, a.head_dim, vf[u]);
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) kf[u][e] = vf[u][e] = 0.f;
            }
        }
        if (VEC && base + kUnroll * kStreams < t1) fetch(base + kUnroll * kStreams);
        float top = m;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            float d[RB];
#pragma unroll
            for (int r = 0; r < RB; ++r) {
                d[r] = 0.f;
#pragma unroll
                for (int e = 0; e < E; ++e) d[r] = fmaf(q[r][e], kf[u][e], d[r]);
            }
            int n = RB;
#pragma unroll
            for (int mask = LPK / 2; mask; mask /= 2) {
                if (n > 1) {
                    n /= 2;
                    const bool up = lane & mask;
#pragma unroll
                    for (int r = 0; r < RB / 2; ++r) {
                        if (r < n) {
                            const float send = up ? d[r] : d[r + n], keep = up ? d[r + n] : d[r];
                            d[r] = keep + __shfl_xor_sync(0xffffffffu, send, mask);
                        }
                    }
                } else {
                    d[0] += __shfl_xor_sync(0xffffffffu, d[0], mask);
                }
            }
            const int32_t j = (int32_t)key[u];
            const bool seen = in[u] && j < mine.hi && (j >= mine.lo || (uint32_t)j < a.sinks);
            s[u] = seen ? d[0] * a.scale : -INFINITY;
            top = fmaxf(top, s[u]);
        }
        const float against = top == -INFINITY ? 0.f : top;
        const float shrink = exp2_approx(m - against);
        m = top;
        l *= shrink;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            s[u] = exp2_approx(s[u] - against) * down;
            l += s[u];
        }
#pragma unroll
        for (int r = 0; r < RB; ++r) {
            const int src = (int)(group * LPK + r * kStep);
            const float f = __shfl_sync(0xffffffffu, shrink, src);
#pragma unroll
            for (int e = 0; e < E; ++e) acc[r][e] *= f;
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const float p = __shfl_sync(0xffffffffu, s[u], src);
                // a key that no query of this row sees leaves nothing behind, whatever its value holds
                if (p != 0.f) {
#pragma unroll
                    for (int e = 0; e < E; ++e) acc[r][e] = fmaf(p, vf[u][e], acc[r][e]);
                }
            }
        }
    }
    // the groups of the warp
    {
        float top = m;
#pragma unroll
        for (int o = LPK; o < 32; o *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float f = m == -INFINITY ? (l != l ? l : 0.f) : exp2_approx(m - top);
        l *= f;
#pragma unroll
        for (int o = LPK; o < 32; o *= 2) l += __shfl_xor_sync(0xffffffffu, l, o);
#pragma unroll
        for (int r = 0; r < RB; ++r) {
            const float fr = __shfl_sync(0xffffffffu, f, (int)(group * LPK + r * kStep));
#pragma unroll
            for (int e = 0; e < E; ++e) {
                float v = fr == 0.f ? 0.f : acc[r][e] * fr;
#pragma unroll
                for (int o = LPK; o < 32; o *= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
                if (group == 0 && c + e < kMostHead) s_acc[warp][r][c + e] = v;
            }
        }
        if (group == 0 && in_key % kStep == 0) {
            s_m[warp][my_row] = top;
            s_l[warp][my_row] = l;
        }
    }
    __syncthreads();
    // the warps of the CTA
    for (uint32_t i = threadIdx.x; i < RB * a.head_dim; i += kThreads) {
        const uint32_t r = i / a.head_dim, col = i - r * a.head_dim;
        float top = s_m[0][r];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) top = fmaxf(top, s_m[w][r]);
        float sum = 0.f, total = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = s_m[w][r] == -INFINITY ? 0.f : exp2_approx(s_m[w][r] - top);
            sum = f == 0.f ? sum : fmaf(s_acc[w][r][col], f, sum);
            total += f == 0.f ? (s_l[w][r] != s_l[w][r] ? s_l[w][r] : 0.f) : s_l[w][r] * f;   // a sum that is no number stays one
        }
        s_acc[0][r][col] = sum;   // read by this thread alone before
        if (col == 0) {
            s_m[kWarps][r] = top;
            s_l[kWarps][r] = total;
        }
    }
    // the CTAs of the cluster
    if (shares > 1) cluster_sync(); else __syncthreads();
    for (uint32_t i = share * kThreads + threadIdx.x; i < n_rows * a.head_dim; i += shares * kThreads) {
        const uint32_t r = i / a.head_dim, col = i - r * a.head_dim;
        float top = -INFINITY, sum = 0.f, total = 0.f;
        if (shares > 1) {
            const uint32_t at_m = smem_u32(&s_m[kWarps][r]), at_l = smem_u32(&s_l[kWarps][r]), at_acc = smem_u32(&s_acc[0][r][col]);
            for (uint32_t k = 0; k < shares; ++k) top = fmaxf(top, load_shared_cluster(map_to_rank(at_m, k)));
            for (uint32_t k = 0; k < shares; ++k) {
                const float mk = load_shared_cluster(map_to_rank(at_m, k)), lk = load_shared_cluster(map_to_rank(at_l, k));
                const float f = mk == -INFINITY ? 0.f : exp2_approx(mk - top);
                if (f != 0.f) sum = fmaf(load_shared_cluster(map_to_rank(at_acc, k)), f, sum);
                total += f == 0.f ? (lk != lk ? lk : 0.f) : lk * f;
            }
        } else {
            sum = s_acc[0][r][col];
            total = s_l[kWarps][r];
        }
        const uint64_t row = r0 + r, qi = row / per_head;
        const uint32_t h = g * per_head + (uint32_t)(row - qi * per_head);
        T* o = static_cast<T*>(a.out) + (int64_t)b * a.out_batch + (int64_t)qi * a.out_token + (int64_t)h * a.out_head;
        o[col] = from_float<T>(total == 0.f ? 0.f : sum / total);
    }
    if (shares > 1) cluster_sync();   // what the others read is read
}

template <typename T, int LPK, int RB>
cudaError_t run(const AttentionArgs& a, int sm_count, cudaStream_t s) {
    const uint64_t rows = (uint64_t)a.queries * (a.heads / a.kv_heads), groups = (rows + RB - 1) / RB;
    const uint64_t items = (uint64_t)a.batch * a.kv_heads * groups;
    uint32_t shares = 1;
    while (shares < 16 && items * shares < 4ull * sm_count && a.keys / (2 * shares) >= 64) shares *= 2;
    if (items * shares > 0x7FFFFFFFull) return cudaErrorInvalidValue;
    auto kernel = attention_rows_kernel<T, LPK, RB, false>;
    if constexpr (RB <= attention_few_rows(sizeof(T))) {
        if (a.vec) kernel = attention_rows_kernel<T, LPK, RB, true>;
    }
    if (shares > 8) {   // clusters of 16 are to be asked for
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((uint32_t)(items * shares));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = shares;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a, (uint32_t)groups);
}

template <typename T, int LPK>
cudaError_t pick_rows(const AttentionArgs& a, int sm_count, cudaStream_t s) {
    const uint64_t rows = (uint64_t)a.queries * (a.heads / a.kv_heads);
    if (rows <= 1) return run<T, LPK, 1>(a, sm_count, s);
    if (rows <= 2) return run<T, LPK, 2>(a, sm_count, s);
    if (rows <= 4) return run<T, LPK, 4>(a, sm_count, s);
    return run<T, LPK, 8>(a, sm_count, s);
}

template <typename T>
cudaError_t pick(const AttentionArgs& a, int sm_count, cudaStream_t s) {
    constexpr uint32_t E = kPer16<T>;
    if (a.head_dim <= 8 * E) return pick_rows<T, 8>(a, sm_count, s);
    if (a.head_dim <= 16 * E) return pick_rows<T, 16>(a, sm_count, s);
    if constexpr (E == 4) return pick_rows<T, 32>(a, sm_count, s);
    return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_attention_rows(const AttentionArgs& a, uint32_t dtype, int sm_count, cudaStream_t s) {
    if (!a.batch || !a.queries || !a.heads) return cudaSuccess;
    return dtype == 0 ? pick<float>(a, sm_count, s) : dtype == 1 ? pick<__half>(a, sm_count, s) : pick<__nv_bfloat16>(a, sm_count, s);
}

}  // namespace lutamm
