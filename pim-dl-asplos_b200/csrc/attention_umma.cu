// Attention for many rows, on the tensor cores:  out = softmax(scale q k^T) v  over the keys that a query sees (attention.cuh).
//
// A CTA takes 128 rows - query tokens times the query heads that share a key head - of one sequence through the keys that any of
// them sees, 64 keys a tile: first the tiles of the sinks, then those of the window; tiles in between are never loaded.  With S = Q K^T
// (tcgen05.mma, queries in tensor memory, keys in shared memory) in tensor memory, a thread owns a row: it reads the 64 scores,
// keeps the running maximum m and sum l, and writes p = exp2(s - m) back over S, where the next product P V reads it as its operand;
// the sum of the tiles' products, rescaled by exp2(m_old - m_new), stays in the thread's registers.  What is exchanged between
// threads is two barriers a tile.  While a tile's weights are formed, the tensor core works on the next tile's scores and the last
// tile's product: S is double, and two CTAs share an SM where head_dim is at most 64.
//
// Types: f16 and bf16 go through as they are; weights are rounded to that type, once, as an operand of the tensor core has to be.
// fp32 operands are split into two f16 numbers, x = hi + lo to 22 bits, and hi hi + hi lo + lo hi is summed; the product of the rests, 2^-22
// of the whole, is left out.  f16 ends at 65504 and thins out below 2^-14, so operands carry a power of two: queries one per row, keys
// and values one per tile, kept from tile to tile for as long as the tile's largest value lies in 1/4 .. 32768 under it; the loading
// warps look at that while they convert, and convert a tile once more where it does not.  Weights carry 2^14, the sum l with
// them.  Maxima, sums and outputs are fp32.
//
// The loading warps read global memory with plain 16-byte loads: no tensor maps, and rows behind the last key become zeros.  Tensors that
// do not start on 16 bytes throughout take the other kernel (attention_rows.cu), element by element.
// Where there are few CTAs, the key tiles of one item are split over a cluster, whose CTAs join through distributed shared memory: no
// scratch memory and one order of summation.
#include "attention.cuh"
#include "ptx.cuh"

#include <algorithm>
#include <type_traits>

namespace lutamm {
namespace {

constexpr int kRows = 128, kKeys = 64, kThreads = 384;
constexpr int kPanel = kKeys * 128;   // bytes: 64 keys x 64 elements of two bytes, swizzled rows of 128 bytes
constexpr uint32_t kMostShares = 8;
// Tensor memory adds up towards zero: a sum of n products is short by about 3e-8 of its size a tile, 1.3e-5 at 16000 keys.  fp32's output is
// taken into registers, where sums are rounded, every so many tiles; half the bits do not show it.
constexpr uint32_t kChunk = 8;
constexpr float kBoost = 6.f, kSlack = 8.f;   // log2 of what weights are multiplied by, and of how far they may grow over 1: 2^14 in all

template <typename T, int DP>
struct Form {
    static constexpr int kParts = sizeof(T) == 4 ? 2 : 1, kPanels = DP / 64;
    static constexpr int kTile = kParts * kPanels * kPanel;          // bytes of a tile of keys or values
    static constexpr int kSlots = 6;                                 // of the ring that keys and values take by turns
    static constexpr int kAhead = 3;                                 // tiles on their way
    static constexpr int kSmem = kSlots * kTile + 1024;
    static constexpr bool kSums = sizeof(T) == 4;                    // sums of products over the tiles in registers: see kChunk
    static constexpr int kScores = 0, kProduct = 2 * kKeys, kQuery = kProduct + DP, kUsed = kQuery + kParts * DP / 2;
    static constexpr int kColumns = kUsed <= 256 ? 256 : 512;
    static constexpr int kCtas = DP <= 64 ? 2 : 1;                   // per SM
    // Registers a thread by role.  Their sum is what the three warpgroups are launched with, 3 x 80 or 3 x 168.
    static constexpr int kRowRegs = DP <= 64 ? 152 : 232, kLoadRegs = DP <= 64 ? 64 : 136, kIssueRegs = DP <= 64 ? 24 : 136;
};
static_assert(152 + 64 + 24 == 3 * 80 && 232 + 136 + 136 == 3 * 168);

template <int N> __device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// kind::f16, fp32 sums, 128 rows: A in tensor memory, two elements a column; B in shared memory.
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
template <typename T>
__device__ __forceinline__ uint32_t idesc_f16(uint32_t n) {
    constexpr uint32_t bf = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return (1u << 4) | (bf << 7) | (bf << 10) | ((n >> 3) << 17) | ((kRows >> 4) << 24);
}
// B whose rows are the contraction axis: 64 elements, one swizzle row of 128 bytes, a row; eight rows a group.
__device__ __forceinline__ uint64_t desc_rows(uint32_t smem_addr) {
    return umma_desc_k_sw128(smem_addr) | (static_cast<uint64_t>(1024u >> 4) << 16);
}

__device__ __forceinline__ void sync_128() { asm volatile("barrier.cta.sync 1, 128;" ::: "memory"); }   // the loading warps
__device__ __forceinline__ float power2(int e) { return __int_as_float((127 + e) << 23); }   // |e| < 127
// The power of two that takes a largest value to 8 .. 16, up to 2^108 (results below 1e-32 have fewer bits); 0 for 0.
__device__ __forceinline__ int exponent_for(uint32_t top_bits) { return top_bits == 0 ? 0 : min(108, 130 - (int)(top_bits >> 23)); }
// Two fp32 operations an instruction.
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// x = hi + lo in f16, two at a time
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
    hi = pack2(a, b, static_cast<__half*>(nullptr));
    const float2 h = unpack2(hi, static_cast<__half*>(nullptr));
    const float2 rest = unpair(fma2(pair(h.x, h.y), pair(-1.f, -1.f), pair(a, b)));
    lo = pack2(rest.x, rest.y, static_cast<__half*>(nullptr));
}
// ... of numbers that may be infinite: their rest is none
__device__ __forceinline__ void split2_any(float a, float b, uint32_t& hi, uint32_t& lo) {
    hi = pack2(a, b, static_cast<__half*>(nullptr));
    const float2 h = unpack2(hi, static_cast<__half*>(nullptr));
    const float x = a - h.x, y = b - h.y;
    lo = pack2(x == x ? x : 0.f, y == y ? y : 0.f, static_cast<__half*>(nullptr));
}

// ones below bit n
__device__ __forceinline__ uint64_t below(int64_t n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1ull; }

struct Bars {
    uint64_t full[6], empty[6], s_full[2], p_full[2], pv_full, all_done, q_full;
};

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, Form<T, DP>::kCtas)
attention_umma_kernel(const __grid_constant__ AttentionArgs a, uint32_t row_tiles, uint32_t* dev_err) {
    using F = Form<T, DP>;
    constexpr uint32_t kSlots = F::kSlots;
    extern __shared__ unsigned char s_raw[];
    __shared__ __align__(8) Bars s_bar;
    __shared__ uint32_t s_tmem, s_abort, s_top[3][4];
    __shared__ int32_t s_exp_k[8], s_exp_v[8];   // by tile: the loading warps are at most three tiles ahead of who reads these
    __shared__ float s_m[kRows], s_l[kRows], s_part[kMostShares][kRows];
    unsigned char* smem = s_raw + ((1024u - (smem_u32(s_raw) & 1023u)) & 1023u);
    const uint32_t smem_at = smem_u32(smem);
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;

    const uint32_t shares = cluster_size_x(), share = cluster_rank();
    uint32_t item = blockIdx.x / shares;
    const uint32_t rt = item % row_tiles;
    item /= row_tiles;
    const uint32_t g = item % a.kv_heads, b = item / a.kv_heads;
    const uint32_t per_head = a.heads / a.kv_heads;
    const uint32_t rows = a.queries * per_head, r0 = rt * kRows;   // below 2^31
    const uint32_t n_rows = min(rows - r0, (uint32_t)kRows);
    const int32_t length = key_count(a, b);
    const int64_t first = a.first ? __ldg(a.first + b) : 0;
    const int64_t p0 = first + r0 / per_head, p1 = first + (r0 + n_rows - 1) / per_head;
    KeySpan span = key_span(a, p0, p1, length);
    if (span.lo <= (span.sinks + kKeys - 1) / kKeys * kKeys) span.lo = span.sinks = 0;   // the window begins in the sinks' last tile
    const uint32_t sink_tiles = (uint32_t)(span.sinks + kKeys - 1) / kKeys;
    const uint32_t all_tiles = sink_tiles + (uint32_t)(((int64_t)span.hi - span.lo + kKeys - 1) / kKeys);
    const uint32_t t0 = (uint32_t)((uint64_t)all_tiles * share / shares), tiles = (uint32_t)((uint64_t)all_tiles * (share + 1) / shares) - t0;
    auto tile_keys = [&](uint32_t j, int32_t& k0, int32_t& end) {
        const uint32_t t = t0 + j;
        const bool sink = t < sink_tiles;
        k0 = sink ? (int32_t)(t * kKeys) : span.lo + (int32_t)((t - sink_tiles) * kKeys);
        end = sink ? span.sinks : span.hi;
    };

    if (warp == 8) {
        tmem_alloc(smem_u32(&s_tmem), F::kColumns);
        tmem_relinquish();
    }
    if (tid == 0) {
        for (int i = 0; i < F::kSlots; ++i) {
            mbar_init(smem_u32(&s_bar.full[i]), 4);
            mbar_init(smem_u32(&s_bar.empty[i]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&s_bar.s_full[i]), 1);
            mbar_init(smem_u32(&s_bar.p_full[i]), 4);
        }
        mbar_init(smem_u32(&s_bar.pv_full), 1);
        mbar_init(smem_u32(&s_bar.all_done), 1);
        mbar_init(smem_u32(&s_bar.q_full), 4);
        fence_barrier_init();
        s_abort = 0;
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = s_tmem;
    const uint32_t dim = a.head_dim;

    auto write_row = [&](uint32_t r, uint32_t c, const float (&w)[4]) {   // four elements from column c
        const uint32_t row = r0 + r, qi = row / per_head, head = g * per_head + (row - qi * per_head);
        T* p = static_cast<T*>(a.out) + (int64_t)b * a.out_batch + (int64_t)qi * a.out_token + (int64_t)head * a.out_head + c;
        if constexpr (sizeof(T) == 4) store_elems<T, 4>(p, w);
        else *reinterpret_cast<uint2*>(p) = make_uint2(pack2(w[0], w[1], static_cast<T*>(nullptr)), pack2(w[2], w[3], static_cast<T*>(nullptr)));
    };
    float4* s_o = reinterpret_cast<float4*>(smem);   // the CTA's part of the result, [row][column / 4], the columns of a row turned

    if (warp < 4) {
        // ---------------------------------------------------------------- a row a thread
        regs_up<F::kRowRegs>();
        const uint32_t lanes = (warp * 32u) << 16;
        const bool real = tid < n_rows;
        const uint32_t row = r0 + (real ? tid : n_rows - 1), qi = row / per_head, head = g * per_head + (row - qi * per_head);
        const KeyBounds mine = key_bounds(a, first + (int64_t)qi, length);
        float factor = fabsf(a.scale), q_up = 1.f;   // of this row's scores; of its query
        {
            const T* qp = static_cast<const T*>(a.q) + (int64_t)b * a.q_batch + (int64_t)qi * a.q_token + (int64_t)head * a.q_head;
            const float sign = a.scale < 0.f ? -1.f : a.scale > 0.f ? 1.f : 0.f;
            if (a.scale == 0.f) factor = 1.f;
            constexpr int E = kPer16<T>;
#pragma unroll
            for (int panel = 0; panel < F::kPanels; ++panel) {   // (fp32: the power of two is the row's, so its largest value comes first)
                uint4 raw[64 / E];
#pragma unroll
                for (int i = 0; i < 64 / E; ++i) {
                    raw[i] = make_uint4(0, 0, 0, 0);
                    if (real && panel * 64u + i * E < dim) raw[i] = __ldg(reinterpret_cast<const uint4*>(qp + panel * 64 + i * E));
                }
                if constexpr (F::kParts == 2) {
                    if (panel == 0) {
                        uint32_t top = 0;
                        auto look = [&](uint32_t bits) {
                            bits &= 0x7FFFFFFFu;
                            if (bits < 0x7F800000u) top = max(top, bits);
                        };
#pragma unroll
                        for (int i = 0; i < 64 / E; ++i) { look(raw[i].x); look(raw[i].y); look(raw[i].z); look(raw[i].w); }
                        if constexpr (F::kPanels == 2) {
#pragma unroll 4
                            for (uint32_t c = 64; c < dim; c += E) {
                                if (real) {
                                    const uint4 w = __ldg(reinterpret_cast<const uint4*>(qp + c));
                                    look(w.x); look(w.y); look(w.z); look(w.w);
                                }
                            }
                        }
                        const int e = exponent_for(top);
                        q_up = power2(e);
                        factor *= power2(-e);
                    }
                }
                const float up = sign * q_up;
#pragma unroll
                for (int part = 0; part < 64 / E / 4; ++part) {   // 4 E elements: 16 columns of 16-bit types, 8 and 8 of fp32
                    if constexpr (F::kParts == 2) {
                        uint32_t hi[8], lo[8];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint4 w = raw[part * 4 + i];
                            split2_any(__uint_as_float(w.x) * up, __uint_as_float(w.y) * up, hi[2 * i], lo[2 * i]);
                            split2_any(__uint_as_float(w.z) * up, __uint_as_float(w.w) * up, hi[2 * i + 1], lo[2 * i + 1]);
                        }
                        tmem_st_32x32b_x8(tmem + lanes + F::kQuery + panel * 32 + part * 8, hi);
                        tmem_st_32x32b_x8(tmem + lanes + F::kQuery + DP / 2 + panel * 32 + part * 8, lo);
                    } else {
                        uint32_t w[16];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t u[4] = {raw[part * 4 + i].x, raw[part * 4 + i].y, raw[part * 4 + i].z, raw[part * 4 + i].w};
#pragma unroll
                            for (int k = 0; k < 4; ++k) w[4 * i + k] = a.scale > 0.f ? u[k] : a.scale < 0.f ? u[k] ^ 0x80008000u : 0u;
                        }
                        tmem_st_32x32b_x16(tmem + lanes + F::kQuery + panel * 32 + part * 16, w);
                    }
                }
            }
            tmem_st_wait();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&s_bar.q_full));
        }
        // All rows see all of a tile that lies between these.
        const int32_t common_hi = key_bounds(a, p0, length).hi, common_lo = key_bounds(a, p1, length).lo;
        float m = -INFINITY, l = 0.f;   // what weights are formed against; their sum, times 2^kBoost
        const uint32_t out_at = tmem + lanes + F::kProduct;
        // fp32: the output of the tiles since the last chunk's end is the one in tensor memory * 2^-unit; that of those before is o, against m_o
        uint64_t o[F::kSums ? DP / 2 : 1];
        float m_o = -INFINITY;
        int unit = 0;
        if constexpr (F::kSums) {
#pragma unroll
            for (int i = 0; i < DP / 2; ++i) o[i] = 0;
        }
        auto add_chunk = [&]() {
            const float against = m == -INFINITY ? 0.f : m, f = exp2_approx(m_o - against), up = power2(-unit);
            const uint64_t f2 = pair(f, f), up2 = pair(up, up);
#pragma unroll
            for (int col = 0; col < DP; col += 16) {
                uint32_t v[16];
                tmem_ld_32x32b_x16(out_at + col, v);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    uint64_t& x = o[col / 2 + i];
                    x = fma2(pair(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), up2, fma2(x, f2, 0ull));
                }
            }
            m_o = m;
        };
        for (uint32_t j = 0; j < tiles; ++j) {
            if (!mbar_wait_warp(smem_u32(&s_bar.s_full[j & 1u]), (j >> 1) & 1u, &s_abort)) break;
            tc_fence_after_sync();
            const uint32_t at = tmem + lanes + F::kScores + (j & 1u) * kKeys;
            bool begun = j > 0;   // whether tensor memory holds an output to go on with
            if constexpr (F::kSums) {
                begun = j % kChunk != 0;
                if (j > 0 && !begun) {
                    if (!mbar_wait_warp(smem_u32(&s_bar.pv_full), (j - 1) & 1u, &s_abort)) break;
                    tc_fence_after_sync();
                    add_chunk();
                }
            }
            float c = factor;
            int e = 0;
            if constexpr (F::kParts == 2) {
                c *= power2(-s_exp_k[j % 8]);
                // the values' power of two is known once they are in shared memory, which the keys' turn does not wait for
                if (!mbar_wait_warp(smem_u32(&s_bar.full[(2 * j + 1) % kSlots]), ((2 * j + 1) / kSlots) & 1u, &s_abort)) break;
                e = s_exp_v[j % 8];
            }
            c = fmaxf(c, 1.17549435e-38f);   // hidden scores, minus infinity, stay that
            int32_t k0, end;
            tile_keys(j, k0, end);
            uint32_t seen0 = 0xFFFFFFFFu, seen1 = 0xFFFFFFFFu;
            const bool edge = !((int64_t)k0 + kKeys <= min(end, common_hi) && (k0 >= common_lo || (int64_t)k0 + kKeys <= (int64_t)a.sinks));
            if (edge) {
                const uint64_t seen = below((int64_t)min(end, mine.hi) - k0) & ~(below((int64_t)mine.lo - k0) & ~below((int64_t)a.sinks - k0));
                seen0 = (uint32_t)seen;
                seen1 = (uint32_t)(seen >> 32);
            }
            auto read = [&](uint32_t (&sc)[32], int half) {
                tmem_ld_32x32b_x32(at + half * 32, sc);
            };
            auto hide = [&](uint32_t (&sc)[32], uint32_t bits) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (!(bits >> i & 1u)) sc[i] = 0xFF800000u;
            };
            auto largest = [&](const uint32_t (&sc)[32]) {
                float t[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                    t[0] = max3(t[0], __uint_as_float(sc[i]), __uint_as_float(sc[i + 1]));
                    t[1] = max3(t[1], __uint_as_float(sc[i + 2]), __uint_as_float(sc[i + 3]));
                }
                return fmaxf(t[0], t[1]);
            };
            uint32_t s0[32], s1[32];
            read(s0, 0);
            read(s1, 1);
            tmem_ld_wait();
            if (edge) {
                hide(s0, seen0);
                hide(s1, seen1);
            }
            const float top = fmaxf(largest(s0), largest(s1)) * c;
            // Another maximum, or another power of two of the values: the output so far is brought in line, where there is one.
            float more = kBoost;   // log2 of what this tile's weights carry
            if (m == -INFINITY) m = top;
            if (!begun || m == -INFINITY) unit = e;
            if (__any_sync(0xffffffffu, top > m + kSlack || unit != e)) {
                const float m_new = top > m + kSlack ? top : m;
                const float shrink = m == -INFINITY ? 1.f : exp2_approx(m - m_new);
                if (begun) {
                    if (!mbar_wait_warp(smem_u32(&s_bar.pv_full), (j - 1) & 1u, &s_abort)) break;
                    tc_fence_after_sync();
                    float f = shrink;
                    if constexpr (F::kParts == 2) {
                        float big = 0.f;
#pragma unroll 1
                        for (uint32_t col = 0; col < DP; col += 16) {
                            uint32_t v[16];
                            tmem_ld_32x32b_x16(out_at + col, v);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 16; ++i) big = fmaxf(big, fabsf(__uint_as_float(v[i])));
                        }
                        // Not to where the output would overflow: then this tile's weights carry the difference, which leaves them without weight.
                        const int x = max(-120, min(120, e - unit));
                        if (x <= 0 || big * shrink < power2(60 - max(x, 0) / 2) * power2(-((max(x, 0) + 1) / 2))) {
                            f *= power2(x);
                            unit = e;
                        }
                    }
#pragma unroll 1
                    for (uint32_t col = 0; col < DP; col += 16) {
                        uint32_t v[16];
                        tmem_ld_32x32b_x16(out_at + col, v);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
                        tmem_st_32x32b_x16(out_at + col, v);
                    }
                    tmem_st_wait();
                }
                l *= shrink;
                m = m_new;
            }
            const float against = m == -INFINITY ? 0.f : m;
            float back = 1.f;
            if constexpr (F::kParts == 2) {
                const int x = max(-120, unit - e);
                more += (float)x;
                back = power2(-x);
            }
            const uint64_t off = pair(more - against, more - against), cc = pair(c, c);
            uint64_t sum[2] = {0, 0};
            if constexpr (F::kSums) {
                // Here the registers hold o, too: the scores are read once more, half by half.  Weights of 32 keys go where their scores lay,
                // 16 columns of them and 16 of their rests.
#pragma unroll 1
                for (int half = 0; half < 2; ++half) {
                    uint32_t sc[32], hi[16], lo[16];
                    read(sc, half);
                    tmem_ld_wait();
                    if (edge) hide(sc, half ? seen1 : seen0);
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float2 x = unpair(fma2(pair(__uint_as_float(sc[i]), __uint_as_float(sc[i + 1])), cc, off));
                        const float p = exp2_approx(x.x), q = exp2_approx(x.y);
                        sum[i / 2 & 1] = add2(sum[i / 2 & 1], pair(p, q));
                        split2(p, q, hi[i / 2], lo[i / 2]);
                    }
                    tmem_st_32x32b_x16(at + half * 32, hi);
                    tmem_st_32x32b_x16(at + half * 32 + 16, lo);
                }
            } else {
                uint32_t w[32];
                auto weights = [&](const uint32_t (&sc)[32], int to) {
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float2 x = unpair(fma2(pair(__uint_as_float(sc[i]), __uint_as_float(sc[i + 1])), cc, off));
                        const float p = exp2_approx(x.x), q = exp2_approx(x.y);
                        sum[i / 2 & 1] = add2(sum[i / 2 & 1], pair(p, q));
                        w[to + i / 2] = pack2(p, q, static_cast<std::conditional_t<sizeof(T) == 4, __half, T>*>(nullptr));
                    }
                };
                weights(s0, 0);
                weights(s1, 16);
                tmem_st_32x32b_x32(at, w);
            }
            tmem_st_wait();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&s_bar.p_full[j & 1u]));
            const float2 sums = unpair(add2(sum[0], sum[1]));
            l = fmaf(sums.x + sums.y, back, l);
        }
        // A barrier's wait tells a phase from the one before it alone, and here the last two products may be done or under way: a barrier of its own.
        const bool done = tiles > 0 && mbar_wait_warp(smem_u32(&s_bar.all_done), 0, &s_abort);
        tc_fence_after_sync();
        const float norm = shares > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l;
        auto put = [&](uint32_t col, float x0, float x1, float x2, float x3) {   // (a row that sees nothing may hold what others' values left)
            const float x[4] = {norm == 0.f ? 0.f : x0 * norm, norm == 0.f ? 0.f : x1 * norm, norm == 0.f ? 0.f : x2 * norm, norm == 0.f ? 0.f : x3 * norm};
            if (shares > 1) s_o[tid * (DP / 4) + ((col / 4) ^ (tid & (DP / 4 - 1)))] = make_float4(x[0], x[1], x[2], x[3]);   // all products are done: nothing reads the tiles
            else if (real && col < dim) write_row(tid, col, x);
        };
        if constexpr (F::kSums) {
            if (done) add_chunk();
#pragma unroll
            for (int col = 0; col < DP; col += 4) {
                const float2 x = unpair(o[col / 2]), y = unpair(o[col / 2 + 1]);
                put(col, x.x, x.y, y.x, y.y);
            }
        } else {
#pragma unroll 1
            for (uint32_t col = 0; col < DP; col += 16) {
                if (col >= dim) break;
                uint32_t v[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = 0;
                if (done) {
                    tmem_ld_32x32b_x16(out_at + col, v);
                    tmem_ld_wait();
                }
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    put(col + i, __uint_as_float(v[i]), __uint_as_float(v[i + 1]), __uint_as_float(v[i + 2]), __uint_as_float(v[i + 3]));
            }
        }
        s_m[tid] = m;
        s_l[tid] = l;
    } else if (warp < 8) {
        // ---------------------------------------------------------------- keys and values into shared memory
        regs_down<F::kLoadRegs>();
        const uint32_t t = tid - 128;
        constexpr int kPerThread = kKeys * DP / 8 / 128;   // groups of eight elements: of one column, kStepRows rows apart
        constexpr int kPerRow = DP / 8, kStepRows = 128 / kPerRow;
        const uint32_t my_row = t / kPerRow, my_col = t % kPerRow;
        const bool in_dim = my_col * 8 < dim;
        const T* kp = static_cast<const T*>(a.k) + (int64_t)b * a.k_batch + (int64_t)g * a.k_head + (in_dim ? my_col * 8 : 0);
        const T* vp = static_cast<const T*>(a.v) + (int64_t)b * a.v_batch + (int64_t)g * a.v_head + (in_dim ? my_col * 8 : 0);
        const int64_t k_step = a.k_token * kStepRows, v_step = a.v_token * kStepRows;
        // where this thread's first group lies in a tile; the rows of its others differ by multiples of eight, which leaves the swizzle as it is
        const uint32_t place = (my_col / 8) * kPanel + my_row * 128u + (((my_col & 7u) ^ (my_row & 7u)) << 4);
        constexpr uint32_t kPlaceStep = kStepRows * 128;
        const uint32_t jobs = 2 * tiles;   // keys of a tile, values of a tile, ...
        // A job's source: this thread's first group, the step between its groups and how many of the groups hold keys.
        struct Source {
            const T* p;
            int64_t step;
            int n;
        };
        auto source = [&](uint32_t job) -> Source {
            int32_t k0, end;
            tile_keys(job / 2, k0, end);
            const int32_t rows_left = end - k0 - (int32_t)my_row;
            Source s;
            s.n = !in_dim || rows_left <= 0 ? 0 : min(kPerThread, (rows_left + kStepRows - 1) / kStepRows);
            const int64_t key = (int64_t)k0 + my_row;
            s.p = job & 1u ? vp + key * a.v_token : kp + key * a.k_token;
            s.step = job & 1u ? v_step : k_step;
            return s;
        };
        auto slot = [&](uint32_t job) -> uint32_t { return job % kSlots * F::kTile; };
        // No early way out of the loops: the four warps meet at a barrier for every tile of fp32.
        auto copy = [&](uint32_t job) {   // this thread's part of a tile, on its way to the job's slot once that is free
            if (job >= kSlots) mbar_wait_warp(smem_u32(&s_bar.empty[job % kSlots]), (job / kSlots - 1) & 1u, &s_abort);
            const Source from = source(job);
            const uint32_t at = smem_at + slot(job);
#pragma unroll
            for (int i = 0; i < kPerThread; ++i) {
                const bool in = i < from.n;
                const T* p = in ? from.p + i * from.step : kp;
#pragma unroll
                for (int h = 0; h < F::kParts; ++h) {   // fp32: two pieces of 16 bytes, to where this thread alone reads them
                    const uint32_t to = F::kParts == 2 ? at + (i * 2 + h) * 2048 + t * 16 : at + place + i * kPlaceStep;
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(in ? p + h * 4 : kp), "r"(in ? 16 : 0) : "memory");
                }
            }
        };
        auto publish = [&](uint32_t job) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&s_bar.full[job % kSlots]));
        };
        // The largest of all loading threads' bits, by turns in three places: a warp is at most one tile ahead of another.
        auto tile_top = [&](uint32_t top, uint32_t turn) -> uint32_t {
            top = __reduce_max_sync(0xffffffffu, top);
            if (lane == 0) s_top[turn][warp - 4] = top;
            sync_128();
            return max(max(s_top[turn][0], s_top[turn][1]), max(s_top[turn][2], s_top[turn][3]));
        };
        int exp_k = 0, exp_v = 0;
        for (uint32_t job = 0; job < F::kAhead; ++job) {
            if (job < jobs) copy(job);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        for (uint32_t job = 0; job < jobs; ++job) {
            if (job + F::kAhead < jobs) copy(job + F::kAhead);
            asm volatile("cp.async.commit_group;" ::: "memory");
            asm volatile("cp.async.wait_group %0;" ::"n"(F::kAhead) : "memory");
            if constexpr (F::kParts == 2) {   // in place, from what this thread has copied itself
                unsigned char* at = smem + slot(job);
                float buf[kPerThread][8];
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < kPerThread; ++i) {
                    const float4 x = *reinterpret_cast<const float4*>(at + (i * 2) * 2048 + t * 16), y = *reinterpret_cast<const float4*>(at + (i * 2 + 1) * 2048 + t * 16);
                    buf[i][0] = x.x; buf[i][1] = x.y; buf[i][2] = x.z; buf[i][3] = x.w;
                    buf[i][4] = y.x; buf[i][5] = y.y; buf[i][6] = y.z; buf[i][7] = y.w;
#pragma unroll
                    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(buf[i][e]) & 0x7FFFFFFFu);
                }
                top = tile_top(top, job & 1u);   // behind it everybody has read
                // 0, or 2^-2 .. 2^15 under the power of two in use, or the tile gets one of its own.
                int& e_now = job & 1u ? exp_v : exp_k;
                const int reach = (int)(top >> 23) - 127 + e_now;
                if (top != 0 && (reach >= 15 || reach < -2)) {
                    if (top >= 0x7F800000u) {   // the largest that is a number
                        uint32_t big = 0;
#pragma unroll
                        for (int i = 0; i < kPerThread; ++i)
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const uint32_t bits = __float_as_uint(buf[i][e]) & 0x7FFFFFFFu;
                                if (bits < 0x7F800000u) big = max(big, bits);
                            }
                        big = tile_top(big, 2);
                        const int r = (int)(big >> 23) - 127 + e_now;
                        if (big != 0 && (r >= 15 || r < -2)) e_now = exponent_for(big);
                    } else {
                        e_now = exponent_for(top);
                    }
                }
                const float up = power2(e_now);
                unsigned char* to = at + place;
#pragma unroll
                for (int i = 0; i < kPerThread; ++i) {
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (top >= 0x7F800000u) split2_any(buf[i][2 * e] * up, buf[i][2 * e + 1] * up, hi[e], lo[e]);
                        else split2(buf[i][2 * e] * up, buf[i][2 * e + 1] * up, hi[e], lo[e]);
                    }
                    *reinterpret_cast<uint4*>(to + i * kPlaceStep) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    *reinterpret_cast<uint4*>(to + i * kPlaceStep + F::kPanels * kPanel) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
                if (t == 0) (job & 1u ? s_exp_v : s_exp_k)[job / 2 % 8] = e_now;
            }
            publish(job);
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    } else {
        // ---------------------------------------------------------------- the tensor core's instructions
        regs_down<F::kIssueRegs>();
        if (warp == 8 && tiles > 0) {
            const uint32_t k_steps = (dim + 15) / 16;
            auto scores = [&](uint32_t j) {   // S = Q K^T, the small products first
                const uint32_t d = tmem + F::kScores + (j & 1u) * kKeys, at = smem_at + 2 * j % kSlots * F::kTile;
                const uint32_t idesc = idesc_f16<T>(kKeys);
                uint32_t more = 0;
#pragma unroll
                for (int term = F::kParts == 2 ? 0 : 2; term < 3; ++term) {
                    const uint32_t qa = tmem + F::kQuery + (term == 1 ? DP / 2 : 0);
                    const uint32_t kb = at + (term == 0 ? F::kPanels * kPanel : 0);
                    for (uint32_t s = 0; s < k_steps; ++s) {
                        umma_f16_ts(d, qa + s * 8, umma_desc_k_sw128(kb + (s / 4) * kPanel + (s % 4) * 32), idesc, more);
                        more = 1;
                    }
                }
            };
            auto product = [&](uint32_t j) {
                const uint32_t p = tmem + F::kScores + (j & 1u) * kKeys, at = smem_at + (2 * j + 1) % kSlots * F::kTile;
#pragma unroll
                for (int panel = 0; panel < F::kPanels; ++panel) {
                    const uint32_t left = dim - panel * 64u, n = left >= 64 ? 64 : (left + 15) / 16 * 16;
                    const uint32_t idesc = idesc_f16<T>(n) | kIdescColumnMajorB;
                    uint32_t more = F::kSums ? j % kChunk != 0 : j > 0;
#pragma unroll
                    for (int term = F::kParts == 2 ? 0 : 2; term < 3; ++term) {
                        const uint32_t pa = p + (term == 1 ? 16 : 0), vb = at + (term == 0 ? F::kPanels * kPanel : 0) + panel * kPanel;
#pragma unroll
                        for (uint32_t s = 0; s < 4; ++s) {
                            umma_f16_ts(tmem + F::kProduct + panel * 64, pa + (F::kParts == 2 ? s / 2 * 32 + s % 2 * 8 : s * 8), desc_rows(vb + s * 2048), idesc, more);
                            more = 1;
                        }
                    }
                }
            };
            bool ok = mbar_wait_warp(smem_u32(&s_bar.q_full), 0, &s_abort);
            ok = ok && mbar_wait_warp(smem_u32(&s_bar.full[0]), 0, &s_abort);
            if (ok) {
                tc_fence_after_sync();
                if (elect_one()) {
                    scores(0);
                    umma_commit(smem_u32(&s_bar.s_full[0]));
                    umma_commit(smem_u32(&s_bar.empty[0]));
                }
                __syncwarp();
            }
            for (uint32_t j = 0; ok && j < tiles; ++j) {
                if (j + 1 < tiles) {
                    // the next tile's scores go where the weights of the tile before this one lie: its product has to be done
                    if (j > 0) ok = mbar_wait_warp(smem_u32(&s_bar.pv_full), (j - 1) & 1u, &s_abort);
                    ok = ok && mbar_wait_warp(smem_u32(&s_bar.full[(2 * j + 2) % kSlots]), ((2 * j + 2) / kSlots) & 1u, &s_abort);
                    if (!ok) break;
                    tc_fence_after_sync();
                    if (elect_one()) {
                        scores(j + 1);
                        umma_commit(smem_u32(&s_bar.s_full[(j + 1) & 1u]));
                        umma_commit(smem_u32(&s_bar.empty[(2 * j + 2) % kSlots]));
                    }
                    __syncwarp();
                }
                ok = mbar_wait_warp(smem_u32(&s_bar.p_full[j & 1u]), (j >> 1) & 1u, &s_abort);
                ok = ok && mbar_wait_warp(smem_u32(&s_bar.full[(2 * j + 1) % kSlots]), ((2 * j + 1) / kSlots) & 1u, &s_abort);
                if (!ok) break;
                tc_fence_after_sync();
                if (elect_one()) {
                    product(j);
                    umma_commit(smem_u32(&s_bar.pv_full));
                    if (j + 1 == tiles) umma_commit(smem_u32(&s_bar.all_done));
                    umma_commit(smem_u32(&s_bar.empty[(2 * j + 1) % kSlots]));
                }
                __syncwarp();
            }
        }
    }

    if (shares > 1) {
        cluster_sync();
        if (tid < n_rows) {   // what each part of a row counts for in the result
            float mk[kMostShares], lk[kMostShares], top = -INFINITY, total = 0.f;
#pragma unroll
            for (uint32_t k = 0; k < kMostShares; ++k) {
                mk[k] = k < shares ? load_shared_cluster(map_to_rank(smem_u32(&s_m[tid]), k)) : -INFINITY;
                lk[k] = k < shares ? load_shared_cluster(map_to_rank(smem_u32(&s_l[tid]), k)) : 0.f;
                top = fmaxf(top, mk[k]);
            }
#pragma unroll
            for (uint32_t k = 0; k < kMostShares; ++k) {
                mk[k] = mk[k] == -INFINITY ? 0.f : exp2_approx(mk[k] - top);
                total += mk[k] == 0.f ? (lk[k] != lk[k] ? lk[k] : 0.f) : lk[k] * mk[k];   // a sum that is no number stays one
            }
            const float norm = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
            for (uint32_t k = 0; k < kMostShares; ++k)
                if (k < shares) s_part[k][tid] = mk[k] == 0.f && norm == norm ? 0.f : mk[k] * norm;
        }
        __syncthreads();
        const uint32_t per_row = dim / 4;
        for (uint32_t i = share * kThreads + tid; i < n_rows * per_row; i += shares * kThreads) {
            const uint32_t r = i / per_row, c = i - r * per_row;
            const uint32_t at_o = smem_u32(&s_o[r * (DP / 4) + (c ^ (r & (DP / 4 - 1)))]);
            float4 x[kMostShares];
            float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (uint32_t k = 0; k < kMostShares; ++k)
                if (k < shares) x[k] = load_shared_cluster4(map_to_rank(at_o, k));
#pragma unroll
            for (uint32_t k = 0; k < kMostShares; ++k)
                if (k < shares) {
                    const float f = s_part[k][r];
                    if (f != 0.f) { v[0] = fmaf(x[k].x, f, v[0]); v[1] = fmaf(x[k].y, f, v[1]); v[2] = fmaf(x[k].z, f, v[2]); v[3] = fmaf(x[k].w, f, v[3]); }
                }
            write_row(r, c * 4, v);
        }
        cluster_sync();   // what the others read is read
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    if (warp == 8 && s_abort) {   // what is in flight gets time to end before its columns are handed back
        const long long from = clock64();
        while (clock64() - from < 200000) {}
        if (lane == 0) report_error(dev_err, 7);
    }
    if (warp == 8) tmem_dealloc(tmem, F::kColumns);
}

template <typename T, int DP>
cudaError_t run(const AttentionArgs& a, int sm_count, uint32_t* dev_err, cudaStream_t s) {
    using F = Form<T, DP>;
    static SmemOptIn memo;
    cudaError_t e = allow_smem(memo, attention_umma_kernel<T, DP>, F::kSmem);
    if (e != cudaSuccess) return e;
    const uint64_t rows = (uint64_t)a.queries * (a.heads / a.kv_heads), tiles = (rows + kRows - 1) / kRows;
    const uint64_t items = (uint64_t)a.batch * a.kv_heads * tiles;
    // Keys that a tile of rows sees at most.
    uint64_t keys = a.keys;
    if (a.left >= 0 && a.right >= 0) keys = std::min<uint64_t>(keys, (uint64_t)a.left + a.right + kRows / (a.heads / a.kv_heads) + 1 + a.sinks);
    uint32_t shares = 1;
    while (shares < kMostShares && items * shares * 2 <= (uint64_t)F::kCtas * sm_count && keys >= 2ull * shares * kKeys) shares *= 2;
    if (rows > 0x7FFFFFFFull || items * shares > 0x7FFFFFFFull) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((uint32_t)(items * shares));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = F::kSmem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = shares;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, attention_umma_kernel<T, DP>, a, (uint32_t)tiles, dev_err);
}

template <typename T>
cudaError_t pick(const AttentionArgs& a, int sm_count, uint32_t* dev_err, cudaStream_t s) {
    return a.head_dim <= 64 ? run<T, 64>(a, sm_count, dev_err, s) : run<T, 128>(a, sm_count, dev_err, s);
}

}  // namespace

cudaError_t launch_attention_umma(const AttentionArgs& a, uint32_t dtype, int sm_count, uint32_t* dev_err, cudaStream_t s) {
    if (!a.batch || !a.queries || !a.heads) return cudaSuccess;
    return dtype == 0 ? pick<float>(a, sm_count, dev_err, s) : dtype == 1 ? pick<__half>(a, sm_count, dev_err, s) : pick<__nv_bfloat16>(a, sm_count, dev_err, s);
}

}  // namespace lutamm
