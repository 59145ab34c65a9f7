// Layer norm over the last axis, forward and backward:
//   y = residual + (x - mean) rstd w + b,   rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   with xh = (x - mean) rstd and g = dy w:  dx = rstd (g - mean(g) - xh mean(g xh)),  dw = sum_rows dy xh,  db = sum_rows dy
//
// All of it is bound by memory: 3 (2 without residual) and 3 times the tensor.  A row is held in registers between its one read
// and its one write, by one to sixteen warps, 16 bytes a load; rows longer than that are read again.  Where a row's start or
// length is no multiple of 16 bytes, loads are of one element, next to one another across the threads.
// 12608 rows of 768 fp32 with the residual 20.1 us, 5.8 TB/s; 128 of them 2.7 us, a launch and two trips to memory.  Backward, 32768 rows
// of 1024 fp32: 71.0 us, 5.7 TB/s; 1576 rows of 1999 bf16: 12.9 us, 1.5 TB/s, loads of two bytes and four rows a CTA.
// Sums are fp32, first over a thread's elements, then pairwise over threads; the variance is the second sum over the registers,
// around the mean.  The gradients of w and b are summed in registers over the rows that a CTA walks, its warps' sums joined
// in shared memory, the CTAs' in a second launch: always in one order, so equal calls give equal bits.
#include "dense.cuh"
#include "kernels.h"

#include <algorithm>
#include <type_traits>

namespace lutamm {
namespace {

constexpr int kMostElems = 8192;   // elements of a row that registers hold in the backward pass

// Sums of a row's threads: TPR of them, all of one warp, or the whole CTA.
template <int TPR, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float (*s)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
    if constexpr (TPR > 32) {
        const uint32_t warp = threadIdx.x >> 5;
        __syncthreads();   // the last sums are read
        if ((threadIdx.x & 31u) == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) s[warp][i] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = 0.f;
#pragma unroll
            for (int w = 0; w < TPR / 32; ++w) v[i] += s[w][i];
        }
    }
}

// One element group of a parameter vector (fp32, any alignment): `missing` where there is none.
template <int E>
__device__ __forceinline__ void load_param(const float* p, bool vec, uint32_t c, float missing, float (&v)[E]) {
    if (!p) {
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = missing;
    } else if (E >= 4 && vec) {
#pragma unroll
        for (int i = 0; i < E / 4; ++i) {
            const float4 f = __ldg(reinterpret_cast<const float4*>(p + c) + i);
            v[4 * i] = f.x; v[4 * i + 1] = f.y; v[4 * i + 2] = f.z; v[4 * i + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = __ldg(p + c + i);
    }
}

template <int TPR> constexpr int kBlock = TPR == 32 ? 256 : TPR;

// A row in registers: NV groups of E elements a thread.
template <typename T, int TPR, int NV, int E>
__global__ void __launch_bounds__(kBlock<TPR>) norm_kernel(NormArgs a) {
    __shared__ float s_sum[TPR / 32][1];
    const uint32_t t = TPR == 32 ? threadIdx.x & 31u : threadIdx.x;
    const uint32_t row = TPR == 32 ? blockIdx.x * (kBlock<TPR> / 32) + (threadIdx.x >> 5) : blockIdx.x;
    if (row >= a.rows) return;   // a warp's row, or the CTA's: no thread waits for one that left
    const T* x = static_cast<const T*>(a.x) + (int64_t)row * a.x_stride;
    const T* r = a.residual ? static_cast<const T*>(a.residual) + (int64_t)row * a.residual_stride : nullptr;
    T* y = static_cast<T*>(a.out) + (int64_t)row * a.out_stride;
    const uint32_t groups = a.width / E;
    float v[NV][E], add[NV][E];
    float sum[1] = {0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const uint32_t g = t + k * TPR;
#pragma unroll
        for (int i = 0; i < E; ++i) v[k][i] = add[k][i] = 0.f;
        if (g < groups) load_elems<T, E>(x + g * E, v[k]);
    }
    if (r) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const uint32_t g = t + k * TPR;
            if (g < groups) load_elems<T, E>(r + g * E, add[k]);
        }
    }
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < E; ++i) sum[0] += v[k][i];
    row_sum<TPR, 1>(sum, s_sum);
    const float mean = sum[0] / (float)a.width;
    sum[0] = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
        if (t + k * TPR < groups) {
#pragma unroll
            for (int i = 0; i < E; ++i) {
                v[k][i] -= mean;
                sum[0] = fmaf(v[k][i], v[k][i], sum[0]);
            }
        }
    row_sum<TPR, 1>(sum, s_sum);
    const float rstd = rsqrtf(sum[0] / (float)a.width + a.eps);
    if (a.stats && t == 0) {
        a.stats[2 * (size_t)row] = mean;
        a.stats[2 * (size_t)row + 1] = rstd;
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const uint32_t g = t + k * TPR;
        if (g < groups) {
            float w[E], b[E], o[E];
            load_param<E>(a.weight, a.param_vec, g * E, 1.f, w);
            load_param<E>(a.bias, a.param_vec, g * E, 0.f, b);
#pragma unroll
            for (int i = 0; i < E; ++i) o[i] = fmaf(v[k][i] * rstd, w[i], b[i]) + add[k][i];
            store_elems<T, E>(y + g * E, o);
        }
    }
}

// Any length: the row is read three times, the second and third from L2 or L1.
template <typename T, int E>
__global__ void __launch_bounds__(512) norm_long_kernel(NormArgs a) {
    __shared__ float s_sum[16][1];
    const uint32_t row = blockIdx.x, groups = a.width / E;
    const T* x = static_cast<const T*>(a.x) + (int64_t)row * a.x_stride;
    const T* r = a.residual ? static_cast<const T*>(a.residual) + (int64_t)row * a.residual_stride : nullptr;
    T* y = static_cast<T*>(a.out) + (int64_t)row * a.out_stride;
    float sum[1] = {0.f};
    for (uint32_t g = threadIdx.x; g < groups; g += 512) {
        float v[E];
        load_elems<T, E>(x + (size_t)g * E, v);
#pragma unroll
        for (int i = 0; i < E; ++i) sum[0] += v[i];
    }
    row_sum<512, 1>(sum, s_sum);
    const float mean = sum[0] / (float)a.width;
    sum[0] = 0.f;
    for (uint32_t g = threadIdx.x; g < groups; g += 512) {
        float v[E];
        load_elems<T, E>(x + (size_t)g * E, v);
#pragma unroll
        for (int i = 0; i < E; ++i) sum[0] = fmaf(v[i] - mean, v[i] - mean, sum[0]);
    }
    row_sum<512, 1>(sum, s_sum);
    const float rstd = rsqrtf(sum[0] / (float)a.width + a.eps);
    if (a.stats && threadIdx.x == 0) {
        a.stats[2 * (size_t)row] = mean;
        a.stats[2 * (size_t)row + 1] = rstd;
    }
    for (uint32_t g = threadIdx.x; g < groups; g += 512) {
        float v[E], add[E], w[E], b[E], o[E];
        load_elems<T, E>(x + (size_t)g * E, v);
#pragma unroll
        for (int i = 0; i < E; ++i) add[i] = 0.f;
        if (r) load_elems<T, E>(r + (size_t)g * E, add);
        load_param<E>(a.weight, a.param_vec, g * E, 1.f, w);
        load_param<E>(a.bias, a.param_vec, g * E, 0.f, b);
#pragma unroll
        for (int i = 0; i < E; ++i) o[i] = fmaf((v[i] - mean) * rstd, w[i], b[i]) + add[i];
        store_elems<T, E>(y + (size_t)g * E, o);
    }
}

// dx of the rows that this CTA walks, and their sums towards dw and db into partial[CTA][2][width].
template <typename T, int TPR, int NV, int E>
__global__ void __launch_bounds__(kBlock<TPR>) norm_grad_kernel(NormGradArgs a) {
    constexpr int kRows = kBlock<TPR> / TPR;   // at a time
    __shared__ float s_sum[TPR / 32][2];
    extern __shared__ float s_part[];   // [2][width]
    const uint32_t t = TPR == 32 ? threadIdx.x & 31u : threadIdx.x, sub = TPR == 32 ? threadIdx.x >> 5 : 0;
    const uint32_t groups = a.width / E;
    float dw[NV][E], db[NV][E];
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < E; ++i) dw[k][i] = db[k][i] = 0.f;
    // The next row's loads are on their way while this one is worked on.
    Piece<T, E> x_raw[NV], d_raw[NV];
    auto fetch = [&](uint64_t row) {
        const T* x = static_cast<const T*>(a.x) + (int64_t)row * a.x_stride;
        const T* dy = static_cast<const T*>(a.dout) + (int64_t)row * a.dout_stride;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const uint32_t g = t + k * TPR;
            if (g < groups) {
                x_raw[k].load(x + g * E);
                d_raw[k].load(dy + g * E);
            }
        }
    };
    const uint64_t first = (uint64_t)blockIdx.x * kRows + sub, step = (uint64_t)gridDim.x * kRows;
    if (first < a.rows) fetch(first);
    for (uint64_t row = first; row < a.rows; row += step) {
        float xh[NV][E], d[NV][E];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            x_raw[k].widen(xh[k]);
            d_raw[k].widen(d[k]);
        }
        if (row + step < a.rows) fetch(row + step);
        const float mean = __ldg(a.stats + 2 * row), rstd = __ldg(a.stats + 2 * row + 1);
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const uint32_t g = t + k * TPR;
            if (g < groups) {
                float w[E];
                load_param<E>(a.weight, a.param_vec, g * E, 1.f, w);
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    xh[k][i] = (xh[k][i] - mean) * rstd;
                    dw[k][i] = fmaf(d[k][i], xh[k][i], dw[k][i]);
                    db[k][i] += d[k][i];
                    d[k][i] *= w[i];
                    sum[0] += d[k][i];
                    sum[1] = fmaf(d[k][i], xh[k][i], sum[1]);
                }
            }
        }
        if (a.dx) {
            row_sum<TPR, 2>(sum, s_sum);
            const float m0 = sum[0] / (float)a.width, m1 = sum[1] / (float)a.width;
            T* dx = static_cast<T*>(a.dx) + (int64_t)row * a.dx_stride;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const uint32_t g = t + k * TPR;
                if (g < groups) {
                    float o[E];
#pragma unroll
                    for (int i = 0; i < E; ++i) o[i] = rstd * (d[k][i] - m0 - xh[k][i] * m1);
                    store_elems<T, E>(dx + g * E, o);
                }
            }
        }
    }
    if (!a.partial) return;
    cudaTriggerProgrammaticLaunchCompletion();   // the join may be set up from here on
    float* out = a.partial + (size_t)blockIdx.x * 2 * a.width;
    if constexpr (kRows == 1) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const uint32_t g = t + k * TPR;
            if (g < groups)
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    out[g * E + i] = dw[k][i];
                    out[a.width + g * E + i] = db[k][i];
                }
        }
    } else {
        for (int w = 0; w < kRows; ++w) {   // one warp after the other: one order
            if (sub == w) {
#pragma unroll
                for (int k = 0; k < NV; ++k) {
                    const uint32_t g = t + k * TPR;
                    if (g < groups)
#pragma unroll
                        for (int i = 0; i < E; ++i) {
                            float* p = s_part + g * E + i;
                            p[0] = w ? p[0] + dw[k][i] : dw[k][i];
                            p[a.width] = w ? p[a.width] + db[k][i] : db[k][i];
                        }
                }
            }
            __syncthreads();
        }
        for (uint32_t c = threadIdx.x; c < 2 * a.width; c += kBlock<TPR>) out[c] = s_part[c];
    }
}

// Any length: dx alone, a row a CTA, read twice; and, before it, ...
template <typename T, int E>
__global__ void __launch_bounds__(512) norm_grad_long_kernel(NormGradArgs a) {
    __shared__ float s_sum[16][2];
    const uint32_t row = blockIdx.x, groups = a.width / E;
    const T* x = static_cast<const T*>(a.x) + (int64_t)row * a.x_stride;
    const T* dy = static_cast<const T*>(a.dout) + (int64_t)row * a.dout_stride;
    T* dx = static_cast<T*>(a.dx) + (int64_t)row * a.dx_stride;
    const float mean = a.stats[2 * (size_t)row], rstd = a.stats[2 * (size_t)row + 1];
    float sum[2] = {0.f, 0.f};
    for (uint32_t g = threadIdx.x; g < groups; g += 512) {
        float v[E], d[E], w[E];
        load_elems<T, E>(x + (size_t)g * E, v);
        load_elems<T, E>(dy + (size_t)g * E, d);
        load_param<E>(a.weight, a.param_vec, g * E, 1.f, w);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            sum[0] += d[i] * w[i];
            sum[1] = fmaf(d[i] * w[i], (v[i] - mean) * rstd, sum[1]);
        }
    }
    row_sum<512, 2>(sum, s_sum);
    const float m0 = sum[0] / (float)a.width, m1 = sum[1] / (float)a.width;
    for (uint32_t g = threadIdx.x; g < groups; g += 512) {
        float v[E], d[E], w[E], o[E];
        load_elems<T, E>(x + (size_t)g * E, v);
        load_elems<T, E>(dy + (size_t)g * E, d);
        load_param<E>(a.weight, a.param_vec, g * E, 1.f, w);
#pragma unroll
        for (int i = 0; i < E; ++i) o[i] = rstd * (d[i] * w[i] - m0 - (v[i] - mean) * rstd * m1);
        store_elems<T, E>(dx + (size_t)g * E, o);
    }
}
// ... the sums over rows, a column a thread, row block blockIdx.y.
template <typename T>
__global__ void __launch_bounds__(256) norm_columns_kernel(NormGradArgs a) {
    const uint32_t c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.width) return;
    float dw = 0.f, db = 0.f;
    for (uint64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float d = to_float(static_cast<const T*>(a.dout)[(int64_t)row * a.dout_stride + c]);
        const float v = to_float(static_cast<const T*>(a.x)[(int64_t)row * a.x_stride + c]);
        dw = fmaf(d, (v - __ldg(a.stats + 2 * row)) * __ldg(a.stats + 2 * row + 1), dw);
        db += d;
    }
    a.partial[(size_t)blockIdx.y * 2 * a.width + c] = dw;
    a.partial[(size_t)blockIdx.y * 2 * a.width + a.width + c] = db;
}

// partial[parts][2][width] -> dw, db: 32 columns a CTA, 32 threads to a column, their sums joined in order.
__global__ void __launch_bounds__(1024) norm_join_kernel(const float* partial, uint32_t parts, uint32_t width, float* dweight, float* dbias) {
    __shared__ float s[32][33];
    const uint32_t lane = threadIdx.x & 31u, k = threadIdx.x >> 5;
    cudaGridDependencySynchronize();   // the partial sums are there
    const uint64_t c = (uint64_t)blockIdx.x * 32 + lane, columns = 2 * (uint64_t)width;
    float sum = 0.f;
    if (c < columns) {
#pragma unroll 8
        for (uint32_t p = k; p < parts; p += 32) sum += partial[(size_t)p * columns + c];
    }
    s[k][lane] = sum;
    __syncthreads();
    sum = warp_sum(s[lane][k]);   // column k of the CTA's
    const uint64_t mine = (uint64_t)blockIdx.x * 32 + k;
    if (lane == 0 && mine < columns) {
        float* out = mine < width ? dweight : dbias;
        if (out) out[mine < width ? mine : mine - width] = sum;
    }
}

bool vec_ok(const void* p, int64_t stride, size_t size) {
    return !p || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && (uint64_t)stride * size % 16 == 0);
}

// Two groups of a row a thread, for which a row gets as many warps as it takes (12608 rows of 768 fp32 with six groups a thread, a warp a row: 22.7 us,
// three 20.7, two 20.1, one 21.5).  Rows of elements that lie apart have up to sixteen of these a thread.
template <typename T, int E>
cudaError_t run_norm(const NormArgs& a, cudaStream_t s) {
    const uint32_t groups = a.width / E, rows8 = (a.rows + 7) / 8;
    if constexpr (E > 1) {
        if (groups <= 32) norm_kernel<T, 32, 1, E><<<rows8, 256, 0, s>>>(a);
        else if (groups <= 64) norm_kernel<T, 32, 2, E><<<rows8, 256, 0, s>>>(a);
        else if (groups <= 128) norm_kernel<T, 64, 2, E><<<a.rows, 64, 0, s>>>(a);
        else if (groups <= 192) norm_kernel<T, 96, 2, E><<<a.rows, 96, 0, s>>>(a);
        else if (groups <= 256) norm_kernel<T, 128, 2, E><<<a.rows, 128, 0, s>>>(a);
        else if (groups <= 512) norm_kernel<T, 256, 2, E><<<a.rows, 256, 0, s>>>(a);
        else if (groups <= 2048) norm_kernel<T, 512, 4, E><<<a.rows, 512, 0, s>>>(a);
        else norm_long_kernel<T, E><<<a.rows, 512, 0, s>>>(a);
    } else {
        if (groups <= 128) norm_kernel<T, 32, 4, 1><<<rows8, 256, 0, s>>>(a);
        else if (groups <= 1024) norm_kernel<T, 128, 8, 1><<<a.rows, 128, 0, s>>>(a);
        else if (groups <= 2048) norm_kernel<T, 256, 8, 1><<<a.rows, 256, 0, s>>>(a);
        else if (groups <= 8192) norm_kernel<T, 512, 16, 1><<<a.rows, 512, 0, s>>>(a);
        else norm_long_kernel<T, 1><<<a.rows, 512, 0, s>>>(a);
    }
    return cudaGetLastError();
}

template <typename T, int TPR, int NV, int E>
cudaError_t run_grad(const NormGradArgs& a, uint32_t ctas, cudaStream_t s) {
    const int bytes = TPR == 32 ? (int)(2 * a.width * sizeof(float)) : 0;   // at most 2 KB: a warp holds 256 elements
    norm_grad_kernel<T, TPR, NV, E><<<ctas, kBlock<TPR>, bytes, s>>>(a);
    return cudaGetLastError();
}

// Threads of a row, by its width: eight elements a thread, so that the sums of several CTAs' columns fit an SM's registers (1576 rows of 2000 bf16, element
// by element, with sixteen 15.2 us, with eight 13.4); sixteen where a CTA of 512 would not be enough.
inline int grad_threads(uint32_t width) { return width <= 256 ? 32 : width <= 1024 ? 128 : width <= 2048 ? 256 : 512; }

template <typename T, int E>
cudaError_t run_norm_grad(const NormGradArgs& a, uint32_t ctas, cudaStream_t s) {
    constexpr int k4 = (4 + E - 1) / E, k8 = 8 / E, k16 = 16 / E;   // groups that make so many elements a thread
    if (a.width <= 32 * 4 && E <= 4) return run_grad<T, 32, k4, E>(a, ctas, s);
    if (a.width <= 32 * 8) return run_grad<T, 32, k8, E>(a, ctas, s);
    if (a.width <= 128 * 8) return run_grad<T, 128, k8, E>(a, ctas, s);
    if (a.width <= 256 * 8) return run_grad<T, 256, k8, E>(a, ctas, s);
    if (a.width <= 512 * 8) return run_grad<T, 512, k8, E>(a, ctas, s);
    return run_grad<T, 512, k16, E>(a, ctas, s);
}

// The parts that the sums towards dw and db come in: CTAs, or row blocks of the columns' kernel.  Four rows a CTA at least, which halves what the
// second launch reads; at most what the SMs hold at once (32768 rows of 1024 fp32 with four CTAs of four warps on an SM 89 us, six 76, seven 72, eight, of
// which one waits, 95).
uint32_t grad_parts(uint32_t rows, uint32_t width, int sm_count) {
    if (width > kMostElems) return std::max(1u, std::min(rows, (uint32_t)sm_count));
    const int threads = grad_threads(width);
    const uint32_t per = 4 * (threads == 32 ? 8 : 1), sets = (rows + per - 1) / per;
    return std::max(1u, std::min(sets, (uint32_t)sm_count * (threads == 512 ? 2 : threads == 256 ? 4 : 7)));
}

template <typename T>
cudaError_t run_typed_grad(const NormGradArgs& a, int sm_count, cudaStream_t s) {
    const bool vec = a.width % kPer16<T> == 0 && vec_ok(a.x, a.x_stride, sizeof(T)) && vec_ok(a.dout, a.dout_stride, sizeof(T)) &&
                     vec_ok(a.dx, a.dx_stride, sizeof(T));
    const uint32_t parts = grad_parts(a.rows, a.width, sm_count);
    cudaError_t e = cudaSuccess;
    if (a.width > kMostElems) {
        if (a.partial) {   // first: dx may be written over x or dout
            norm_columns_kernel<T><<<dim3((a.width + 255) / 256, parts), 256, 0, s>>>(a);
            e = cudaGetLastError();
        }
        if (e == cudaSuccess && a.dx && a.rows) {
            if (vec) norm_grad_long_kernel<T, kPer16<T>><<<a.rows, 512, 0, s>>>(a);
            else norm_grad_long_kernel<T, 1><<<a.rows, 512, 0, s>>>(a);
            e = cudaGetLastError();
        }
    } else {
        e = vec ? run_norm_grad<T, kPer16<T>>(a, parts, s) : run_norm_grad<T, 1>(a, parts, s);
    }
    if (e != cudaSuccess || !a.partial) return e;
    // The join is set up while the last rows are walked (32768 rows of 1024 fp32 71.9 -> 70.7 us, 1576 of 2000 bf16 15.2 -> 14.6).
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((uint32_t)((2 * (uint64_t)a.width + 31) / 32));
    cfg.blockDim = dim3(1024);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, norm_join_kernel, static_cast<const float*>(a.partial), parts, a.width, a.dweight, a.dbias);
}

}  // namespace

cudaError_t launch_norm(const NormArgs& a, uint32_t dtype, cudaStream_t s) {
    if (!a.rows) return cudaSuccess;
    auto run = [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const bool vec = a.width % kPer16<T> == 0 && vec_ok(a.x, a.x_stride, sizeof(T)) && vec_ok(a.residual, a.residual_stride, sizeof(T)) &&
                         vec_ok(a.out, a.out_stride, sizeof(T));
        return vec ? run_norm<T, kPer16<T>>(a, s) : run_norm<T, 1>(a, s);
    };
    return dtype == 0 ? run(static_cast<float*>(nullptr)) : dtype == 1 ? run(static_cast<__half*>(nullptr)) : run(static_cast<__nv_bfloat16*>(nullptr));
}

size_t norm_grad_workspace(uint32_t rows, uint32_t width, int sm_count) { return (size_t)grad_parts(rows, width, sm_count) * 2 * width * sizeof(float); }

cudaError_t launch_norm_grad(const NormGradArgs& a, uint32_t dtype, int sm_count, cudaStream_t s) {
    if (!a.rows && !a.partial) return cudaSuccess;
    return dtype == 0 ? run_typed_grad<float>(a, sm_count, s) : dtype == 1 ? run_typed_grad<__half>(a, sm_count, s) : run_typed_grad<__nv_bfloat16>(a, sm_count, s);
}
uint32_t norm_grad_launches(const NormGradArgs& a) {
    return (a.width > kMostElems ? (a.dx && a.rows ? 1 : 0) + (a.partial ? 1 : 0) : 1) + (a.partial ? 1 : 0);
}

}  // namespace lutamm
