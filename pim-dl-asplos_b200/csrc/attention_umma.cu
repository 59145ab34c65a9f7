// Attention for two rows and more (query tokens times the heads of a key head), on the tensor cores:  out = softmax(scale q k^T) v  over the keys that a
// query sees (attention.cuh).
//
// A CTA takes 128 rows - query tokens times the query heads that share a key head - or, of fp32, twice 128, of one sequence through the keys that
// any of them sees, 64 keys a tile: first the tiles of the sinks, then those of the window; tiles in between are never loaded.  Scores S = Q K^T
// (tcgen05.mma, queries in tensor memory, keys in shared memory) go to tensor memory, where a thread owns a row: it reads the 64 scores, takes the
// largest, and writes weights p = exp2(s - m) back over S, where the next product P V reads them as its operand; their sum l stays with the thread.  The
// output stays in tensor memory, too, in 16 bits.  It is brought in line, multiplied by exp2(m_old - m), only where a row's maximum has grown by 2^8: until then
// weights are formed against the old m (a published technique, known as lazy or conditional rescaling).  While a tile's weights are formed, the tensor core works on the next tile's scores and the last tile's product.
//
// Types: f16 and bf16 go through as they are, weights as two numbers of that type, the rounded one and what that leaves: results are rounded once, as where one row
// takes the other kernel (rounded weights alone: 2.3e-3 off for 1.7e-3 in bf16, 2.9e-4 for 2.1e-4 in f16; 8192 tokens 103 us for 115 when this was taken).  fp32 operands are split into
// three bf16 numbers, x = a + b + c: a the leading bits, b and c the rests to nearest, together all 24 bits of x and, bf16 having fp32's exponents, whatever
// its size.  Of the nine products the six down to 2^-16 of the whole are summed, the small ones first; b c + c b, 2^-25 of it, is left out.  So an element's
// digits do not hang on its neighbours', as they would under a power of two for a row or a tile, which half the products of f16 parts need.  f16's weights
// carry 2^6 and up to 2^8 more, the sum l with them; in bf16 and fp32 they, or the values, are brought down by the number of keys instead, exactly, so that a
// row's sums stay below its largest value: results up to the type's largest number do not overflow on the way.  Maxima, sums and outputs are fp32; maxima are taken up to whole numbers, so that what is against an older
// one is brought in line without rounding; the sums over tiles, or chunks of them, outside of tensor memory round once each.
//
// Loading warps copy 16 bytes a piece (cp.async): no tensor maps to be made by the host, and rows behind the last key become zeros.  fp32 is
// converted in place.  Tensors that do not start on 16 bytes throughout take the other kernel (attention_rows.cu), element by element.  Where there are few
// CTAs, the key tiles of one item are split over a cluster, whose CTAs join through distributed shared memory: no scratch memory and one order of summation.
//
// Infinities and NaN: a product over 64 keys would have each meet weights of zero, those of rows and warps that do not see its key, and parts of zero.  So values
// that are not finite go into the product as zeros, and are added to the results of the rows that see them at the end; of keys and queries that are not finite fp32
// forms the scores one by one.  A CTA that meets none pays for the look at what it loads.
//
// What bounds it: issuing instructions.  8192 tokens, 16 heads of 64 in bf16, a window of 512 on either side: 118 us, 283 TFLOP/s; of 3690 warp instructions a
// tile 1300 form its weights, 100 look at its values.  The exponentials alone would take 34 us, the products, three for two, 31.  2048 tokens, 8 heads of 128, all keys: 38 us,
// 450 TFLOP/s.  fp32, six products for one: ViT's batch of 64 x 197 tokens, 12 heads, 113 us, issue in 48 % of the cycles, the tensor cores busy in 30 %: each of the two CTAs on
// an SM is a chain of copy, conversion, scores, weights, product and sum, four tiles long.
#include "attention.cuh"
#include "ptx.cuh"

#include <algorithm>
#include <type_traits>

namespace lutamm {
namespace {

constexpr int kRows = 128, kKeys = 64;
constexpr int kPanel = kKeys * 128;   // bytes: 64 keys x 64 elements of two bytes, swizzled rows of 128 bytes
constexpr uint32_t kMostShares = 8;
// Tensor memory adds up towards zero: fp32's product of a tile takes four units of 2^-24 off the sum at most, its small terms being first, and would take
// twenty-four off with the tiles before in there.  So each tile's is taken out and summed with rounding; of 16-bit types, whose tiles take eight units off at most,
// every 64 (400000 keys of one sign in f16 came out 3e-3 too small without).
constexpr float kBoost = 6.f, kSlack = 8.f;   // log2 of what f16's weights are multiplied by, and of how far they may grow over 1: 2^14 in all

// DP: columns of a head, up to a multiple of 64.  RT: tiles of rows of a CTA, which read the same keys and values.
template <typename T, int DP, int RT>
struct Form {
    static constexpr bool kFp32 = sizeof(T) == 4;
    static constexpr int kParts = kFp32 ? 3 : 1, kPanels = DP / 64;
    static constexpr int kPart = kPanels * kPanel, kTile = kParts * kPart;   // bytes of a part of a tile of keys or values, of the tile
    static constexpr int kSlots = !kFp32 ? 8 : RT == 2 ? 6 : 3;              // of the ring that keys and values take by turns
    static constexpr int kAhead = kFp32 ? 1 : 4;                             // tiles that a warpgroup has on their way
    static constexpr int kOut = RT * kRows * DP * 4;                         // bytes of the output, in fp32: queries come, and results leave, through there
    static constexpr int kSmem = kSlots * kTile + kOut + 1024;
    // Columns of tensor memory of a tile of rows: scores, over which its weights are written, kBufs times; the product; the queries.  Where two buffers of scores
    // find no room, the next tile's are formed behind the product, while the other tile of rows, or the other CTA on the SM, has its weights formed.
    static constexpr uint32_t kChunk = kFp32 ? 1 : 64;                       // tiles whose products are summed in tensor memory
    static constexpr int kScoreCols = kFp32 ? 96 : 64, kBufs = kFp32 && DP <= 64 ? 1 : 2;
    static constexpr int kScores = 0, kProduct = kBufs * kScoreCols, kQuery = kProduct + DP, kUsed = kQuery + kParts * DP / 2;
    static constexpr int kColumns = RT * kUsed <= 256 ? 256 : 512;
    static_assert(RT * kUsed <= 512 && (RT == 1 || kUsed <= 256));
    static constexpr int kCtas = DP <= 64 && RT == 1 ? 2 : 1;        // per SM
    // Warpgroups: one for each tile of rows, a row a thread, one for each tile of rows that loads, one that issues.  Registers a thread of each; their sum is
    // what the warpgroups are launched with.  None of 16-bit types and none of few rows spills (the issuing warps did with 24: 24 rows of 8 x 8192 keys in bf16
    // 59.9 us, 54.4 so); fp32's others keep 16 to 48 bytes a thread in memory, with 136 as with 160 registers for a row.
    static constexpr int kRowWarps = 4 * RT, kIssueAt = 8 * RT, kThreads = (2 * RT + 1) * 128;
    static constexpr int kLaunchRegs = DP > 64 ? 168 : RT == 2 ? 96 : 80, kRowRegs = DP > 64 ? 232 : 136, kLoadRegs = DP > 64 ? 136 : RT == 2 ? 80 : 56;
    static constexpr int kIssueRegs = DP > 64 ? 136 : 48;
    static_assert(RT * (kRowRegs + kLoadRegs) + kIssueRegs == (2 * RT + 1) * kLaunchRegs && kCtas * kThreads * kLaunchRegs <= 65536);
};

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
    constexpr uint32_t bf = std::is_same<T, __half>::value ? 0u : 1u;
    return (1u << 4) | (bf << 7) | (bf << 10) | ((n >> 3) << 17) | ((kRows >> 4) << 24);
}
// B whose rows are the contraction axis: 64 elements, one swizzle row of 128 bytes, a row; eight rows a group.
__device__ __forceinline__ uint64_t desc_rows(uint32_t smem_addr) {
    return umma_desc_k_sw128(smem_addr) | (static_cast<uint64_t>(1024u >> 4) << 16);
}

__device__ __forceinline__ float power2(int e) { return __int_as_float((127 + e) << 23); }   // |e| < 127
__device__ __forceinline__ void sync_128(uint32_t id) { asm volatile("barrier.cta.sync %0, 128;" ::"r"(id) : "memory"); }
// A warp's bounded wait, with one answer.  The hint lets the hardware hold a waiting warp for up to two microseconds a look: without it the fifteen warps
// of a CTA that wait for one another took a third of all instructions.
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, volatile uint32_t* abort_word) {
    uint32_t ok = 0;
    for (uint32_t it = 0; it < 1u << 18; ++it) {
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok) : "r"(bar), "r"(parity), "r"(2000u) : "memory");
        if (__all_sync(0xffffffffu, ok)) return true;
        if (*abort_word) return false;
    }
    *abort_word = 1u;
    return false;
}

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
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// x = hi + mid + lo in bf16, two at a time: hi cut off, which no finite number makes an infinity of, the others to nearest
__device__ __forceinline__ void split3(float a, float b, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
    hi = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
    const uint64_t minus = pair(-1.f, -1.f);
    const float2 h = unpack2(hi, static_cast<__nv_bfloat16*>(nullptr));
    const float2 rest = unpair(fma2(pair(h.x, h.y), minus, pair(a, b)));
    mid = pack2(rest.x, rest.y, static_cast<__nv_bfloat16*>(nullptr));
    const float2 m = unpack2(mid, static_cast<__nv_bfloat16*>(nullptr));
    const float2 last = unpair(fma2(pair(m.x, m.y), minus, pair(rest.x, rest.y)));
    lo = pack2(last.x, last.y, static_cast<__nv_bfloat16*>(nullptr));
}
// x = hi + lo to nearest, in 16 bits
template <typename T>
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
    hi = pack2(a, b, static_cast<T*>(nullptr));
    const float2 h = unpack2(hi, static_cast<T*>(nullptr));
    const float2 rest = unpair(fma2(pair(h.x, h.y), pair(-1.f, -1.f), pair(a, b)));
    lo = pack2(rest.x, rest.y, static_cast<T*>(nullptr));
}
// 0, or NaN where one of the numbers is none or infinite: what is added to `odd`
__device__ __forceinline__ uint64_t look(const float4& x, uint64_t odd) {
    return fma2(pair(x.x, x.y), pair(0.f, 0.f), fma2(pair(x.z, x.w), pair(0.f, 0.f), odd));
}
__device__ __forceinline__ bool is_odd(uint64_t odd) {
    const float2 v = unpair(odd);
    return v.x + v.y != 0.f;
}
__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }
// The same of two 16-bit numbers
__device__ __forceinline__ __half2 look(uint32_t w, __half2 odd) { return __hfma2(*reinterpret_cast<const __half2*>(&w), __half2half2(__ushort_as_half(0)), odd); }
__device__ __forceinline__ __nv_bfloat162 look(uint32_t w, __nv_bfloat162 odd) {
    return __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&w), __bfloat162bfloat162(__ushort_as_bfloat16(0)), odd);
}
// Zero in place of those that are none or infinite: whose exponents, all ones, carry into bit 15 of their half
template <typename T>
__device__ __forceinline__ uint32_t only_finite(uint32_t w) {
    constexpr bool half = std::is_same<T, __half>::value;
    const uint32_t odd = ((w & (half ? 0x7C007C00u : 0x7F807F80u)) + (half ? 0x04000400u : 0x00800080u)) & 0x80008000u;
    return w & ~((odd >> 15) * 0xFFFFu);
}

// ones below bit n
__device__ __forceinline__ uint64_t below(int64_t n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1ull; }

struct RowBars {   // of a tile of rows
    uint64_t s_full[2], p_full[2], done[2], q_full;   // scores, weights and products of every other tile; queries
};

// Which of the CTA's tiles of keys a tile of rows sees any of: the sinks', and from .. to - 1.
struct Seen {
    uint32_t sink_tiles, from, to;
    __device__ __forceinline__ bool operator()(uint32_t t) const { return t < sink_tiles || (t >= from && t < to); }
};

// n / d for n below 2^31: the quotient's 32 bits above the binary point of n * mul / 2^(31 + shift).
struct Divisor {
    uint32_t d, mul, shift;
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return d == 1 ? n : (uint32_t)(((uint64_t)n * mul) >> shift); }
};
Divisor divisor(uint32_t d) {
    uint32_t bits = 0;
    while ((1ull << bits) < d) ++bits;
    return Divisor{d, (uint32_t)(d == 1 ? 0 : (1ull << (31 + bits)) / d + 1), 31 + bits};
}

// FEW: at most 32 rows.  All four warps of rows have them, each with sixteen keys of every tile and an output of its own; they join in the end.  One warp with
// all 64 keys would have the three others idle: tokens of 16 heads on 4 of 128 behind 8 caches of up to 32768, four rows, 67 us so, 54.5 with four warps (57 with the sums out of tensor memory, 4.7 TB/s).
template <typename T, int DP, int RT, bool FEW>
__global__ void __launch_bounds__(Form<T, DP, RT>::kThreads, Form<T, DP, RT>::kCtas)
attention_umma_kernel(const __grid_constant__ AttentionArgs a, const Divisor row_tiles, const Divisor kv_heads, const Divisor per_head, uint32_t* dev_err) {
    using F = Form<T, DP, RT>;
    static_assert(!FEW || RT == 1);
    constexpr uint32_t kSlots = F::kSlots, kThreads = F::kThreads;
    extern __shared__ unsigned char s_raw[];
    __shared__ __align__(8) uint64_t s_full_bar[kSlots], s_empty_bar[kSlots], s_looked_bar[F::kFp32 ? 1 : kSlots];   // (the last: of 16-bit values)
    __shared__ __align__(8) RowBars s_row[RT];
    __shared__ uint32_t s_tmem, s_abort, s_odd_from[2], s_odd_to[2];   // keys, values that are not finite: in tiles from .. to - 1, so far
    __shared__ float s_m[RT * kRows], s_l[RT * kRows], s_join[FEW ? 2 : 1][32];
    unsigned char* smem = s_raw + ((1024u - (smem_u32(s_raw) & 1023u)) & 1023u);
    const uint32_t smem_at = smem_u32(smem);
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;

    const uint32_t shares = cluster_size_x(), share = cluster_rank();
    uint32_t item = shares == 1 ? blockIdx.x : blockIdx.x / shares;
    const uint32_t ct = item - row_tiles(item) * row_tiles.d;
    item = row_tiles(item);
    const uint32_t b = kv_heads(item), g = item - b * kv_heads.d;
    const uint32_t rows = a.queries * per_head.d, r0 = ct * (RT * kRows);   // below 2^31
    const uint32_t n_rows = min(rows - r0, (uint32_t)(RT * kRows));
    const int32_t length = key_count(a, b);
    const int64_t first = a.first ? __ldg(a.first + b) : 0;
    const uint32_t dim = a.head_dim;
    KeySpan span = key_span(a, first + per_head(r0), first + per_head(r0 + n_rows - 1), length);
    // Where the window begins in the sinks' last tile, the tiles run on from the first key; keys that no row sees are left out of them.
    const int32_t gap_from = span.sinks, gap_to = span.lo;
    if (span.lo <= (span.sinks + kKeys - 1) / kKeys * kKeys) span.lo = span.sinks = 0;
    const uint32_t sink_tiles = (uint32_t)(span.sinks + kKeys - 1) / kKeys;
    const uint32_t all_tiles = sink_tiles + (uint32_t)(span.hi - span.lo + kKeys - 1) / kKeys;
    const int log_keys = all_tiles <= 1 ? 6 : 38 - __clz(all_tiles - 1);   // 2^log_keys: no fewer than the keys of all tiles
    const uint32_t t0 = (uint32_t)((uint64_t)all_tiles * share / shares), t1 = (uint32_t)((uint64_t)all_tiles * (share + 1) / shares), tiles = t1 - t0;
    auto tile_keys = [&](uint32_t t, int32_t& k0, int32_t& end) {
        const bool sink = t < sink_tiles;
        k0 = sink ? (int32_t)(t * kKeys) : span.lo + (int32_t)((t - sink_tiles) * kKeys);
        end = sink ? span.sinks : span.hi;
    };
    auto rows_see = [&](uint32_t rt) -> Seen {   // tile rt of the rows
        Seen v{0, 0, 0};
        if (rt * kRows >= n_rows) return v;
        if (RT == 1) return Seen{sink_tiles, sink_tiles, all_tiles};
        const KeySpan own = key_span(a, first + per_head(r0 + rt * kRows), first + per_head(r0 + min((rt + 1) * kRows, n_rows) - 1), length);
        const int32_t lo = max(own.lo, span.lo), hi = min(own.hi, span.hi);
        if (own.hi <= own.lo && own.sinks == 0) return v;
        v.sink_tiles = sink_tiles;
        v.from = sink_tiles + (own.sinks > 0 && span.lo == 0 ? 0u : (uint32_t)(lo - span.lo) / kKeys);   // sinks within the window's tiles
        v.to = hi > span.lo ? sink_tiles + (uint32_t)(hi - span.lo + kKeys - 1) / kKeys : sink_tiles;
        return v;
    };

    // ---- what loads keys and values: warpgroup wg of them (with two, one loads keys, one values)
    const uint32_t t = tid & 127u, wg = warp / 4 - RT;
    // A thread copies pieces of 16 bytes: of one column, kStepRows rows apart, so that neighbours copy whole rows.
    constexpr int kElems = kPer16<T>, kPerRow = DP / kElems, kStepRows = 128 / kPerRow, kPerThread = kKeys / kStepRows;
    const uint32_t my_row = t / kPerRow, my_col = t % kPerRow * kElems;
    const bool in_dim = my_col < dim;
    // Where this thread's first piece lies in a tile (of fp32: 8 bytes of it); the rows of its others differ by multiples of eight, which leaves the
    // swizzle as it is, or of four, which turns a bit of it every time.
    const uint32_t place = my_col / 64 * kPanel + my_row * 128u + ((my_col / 8 % 8 ^ (my_row & 7u)) << 4) + my_col % 8 * 2;
    auto place_of = [&](int i) -> uint32_t { return (kStepRows == 4 && (i & 1) ? place ^ 64u : place) + i * kStepRows * 128; };
    static_assert(kStepRows == 4 || kStepRows % 8 == 0);
    // Jobs are keys of a tile, values of a tile, and so on; this warpgroup's are every RT-th from wg on.
    const uint32_t jobs = 2 * tiles;
    // No early way out of the loops: the four warps meet at a barrier for every tile of fp32.
    auto copy = [&](uint32_t job) {   // this thread's part of a tile, on its way to the job's slot once that is free
        if (job >= kSlots) wait_warp(smem_u32(&s_empty_bar[job % kSlots]), (job / kSlots - 1) & 1u, &s_abort);
        int32_t k0, end;
        tile_keys(t0 + job / 2, k0, end);
        const bool values = job & 1u;
        const int64_t token = values ? a.v_token : a.k_token;
        const T* base = values ? static_cast<const T*>(a.v) + (int64_t)b * a.v_batch + (int64_t)g * a.v_head
                               : static_cast<const T*>(a.k) + (int64_t)b * a.k_batch + (int64_t)g * a.k_head;
        const T* from = base + (int64_t)(k0 + (int32_t)my_row) * token + (in_dim ? my_col : 0);
        const int64_t step = token * kStepRows;
        const uint32_t at = smem_at + job % kSlots * F::kTile;
        auto to = [&](int i) -> uint32_t { return at + (F::kFp32 ? i * 2048 + t * 16 : place_of(i)); };   // (fp32: to where this thread alone reads it)
        if ((uint32_t)k0 + kKeys <= (uint32_t)end && (k0 >= gap_to || (uint32_t)k0 + kKeys <= (uint32_t)gap_from)) {
            const uint32_t size = in_dim ? 16u : 0u;
#pragma unroll
            for (int i = 0; i < kPerThread; ++i, from += step)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to(i)), "l"(from), "r"(size) : "memory");
        } else {
#pragma unroll
            for (int i = 0; i < kPerThread; ++i, from += step) {
                const int32_t key = k0 + (int32_t)my_row + i * kStepRows;
                const bool in = in_dim && key < end && (key < gap_from || key >= gap_to);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to(i)), "l"(in ? from : base), "r"(in ? 16 : 0) : "memory");
            }
        }
    };

    // The first copies leave before the CTA has met.  Queries go row by row through shared memory, 32 rows a warp, so that loads are of whole
    // lines; then a thread has its own row.
    constexpr int kPerQ = DP / kPer16<T>;   // pieces of 16 bytes a row
    const uint32_t warp_row = warp * 32u, first_row = FEW ? 0u : warp_row, q_stage = kSlots * F::kTile + warp_row * DP * 4;   // where the warp's output goes
    if (warp < F::kRowWarps) {
        const uint32_t c = lane % kPerQ;
        const bool in_row = c * kPer16<T> < dim;
        const T* qb = static_cast<const T*>(a.q) + (int64_t)b * a.q_batch + (int64_t)(g * per_head.d) * a.q_head + (in_row ? c * kPer16<T> : 0);
#pragma unroll 4
        for (uint32_t r = lane / kPerQ; r < 32; r += 32 / kPerQ) {
            const bool in = in_row && first_row + r < n_rows;
            const uint32_t row = r0 + (in ? first_row + r : 0u), qi = per_head(row);
            const T* p = qb + (int64_t)qi * a.q_token + (int64_t)(row - qi * per_head.d) * a.q_head;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_at + q_stage + (r * kPerQ + (c ^ (r & (kPerQ - 1)))) * 16), "l"(p), "r"(in ? 16 : 0) : "memory");
        }
    } else if (warp < F::kIssueAt) {
        for (uint32_t i = 0; i < F::kAhead; ++i) {
            if (wg + i * RT < jobs) copy(wg + i * RT);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
    } else if (warp == F::kIssueAt) {
        tmem_alloc(smem_u32(&s_tmem), F::kColumns);
        tmem_relinquish();
    } else if (warp == F::kIssueAt + 1) {
        if (lane < kSlots) mbar_init(smem_u32(&s_full_bar[lane]), 4);
        if (lane < kSlots) mbar_init(smem_u32(&s_empty_bar[lane]), RT);
        if (!F::kFp32 && lane < kSlots) mbar_init(smem_u32(&s_looked_bar[F::kFp32 ? 0 : lane]), 2);
        if (lane < RT) {
            RowBars& bar = s_row[lane];
            for (int i = 0; i < 2; ++i) {
                mbar_init(smem_u32(&bar.s_full[i]), 1);
                mbar_init(smem_u32(&bar.p_full[i]), 4);
                mbar_init(smem_u32(&bar.done[i]), 1);
            }
            mbar_init(smem_u32(&bar.q_full), 4);
        }
        fence_barrier_init();
        if (lane < 2) {
            s_odd_from[lane] = ~0u;
            s_odd_to[lane] = 0;
        }
        if (lane == 0) s_abort = 0;
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = s_tmem;
    float4* s_o = reinterpret_cast<float4*>(smem + kSlots * F::kTile);   // the CTA's part of the result, [row][column / 4], the columns of a row turned
    auto out_place = [](uint32_t r, uint32_t c4) -> uint32_t { return r * (DP / 4) + (c4 ^ (r & (DP / 4 - 1))); };
    auto row_at = [&](uint32_t r) -> T* {   // where a row goes
        const uint32_t row = r0 + r, qi = per_head(row), head = g * per_head.d + (row - qi * per_head.d);
        return static_cast<T*>(a.out) + (int64_t)b * a.out_batch + (int64_t)qi * a.out_token + (int64_t)head * a.out_head;
    };
    auto write_row = [&](uint32_t r, uint32_t c, const float4& v) {   // four elements from column c
        T* p = row_at(r) + c;
        if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(p) = v;
        else *reinterpret_cast<uint2*>(p) = make_uint2(pack2(v.x, v.y, static_cast<T*>(nullptr)), pack2(v.z, v.w, static_cast<T*>(nullptr)));
    };

    auto add_part = [](float4& v, float& total, const float4& x, float l, float f) {   // a part that counts f times
        if (f != 0.f) { v.x = fmaf(x.x, f, v.x); v.y = fmaf(x.y, f, v.y); v.z = fmaf(x.z, f, v.z); v.w = fmaf(x.w, f, v.w); }
        total += f == 0.f ? (l != l ? l : 0.f) : l * f;   // a sum that is no number stays one
    };

    if (warp < F::kRowWarps) {
        // ---------------------------------------------------------------- a row a thread
        regs_up<F::kRowRegs>();
        const uint32_t rt = warp / 4, lanes = ((warp & 3u) * 32u) << 16, r = warp_row + lane;
        RowBars& bar = s_row[rt];
        const uint32_t my_tmem = tmem + rt * 256u + lanes;
        const uint32_t row = r0 + min(first_row + lane, n_rows - 1), qi = per_head(row);
        const KeyBounds mine = key_bounds(a, first + (int64_t)qi, length);
        const Seen sees = rows_see(rt);
        float factor = fabsf(a.scale);   // of this row's scores
        float up = a.scale < 0.f ? -1.f : a.scale > 0.f ? 1.f : 0.f;   // of this row's queries
        bool odd_queries = false;
        if (a.scale == 0.f) factor = 1.f;
        {
            asm volatile("cp.async.wait_all;" ::: "memory");
            __syncwarp();
            auto raw = [&](int i) -> uint4 { return *reinterpret_cast<const uint4*>(smem + q_stage + (lane * kPerQ + (i ^ (lane & (kPerQ - 1)))) * 16); };
            auto raw4 = [&](int i) -> float4 { const uint4 u = raw(i); return *reinterpret_cast<const float4*>(&u); };
            if constexpr (F::kFp32) {
                uint64_t odd = 0;
                float big = 0.f;
#pragma unroll
                for (int i = 0; i < kPerQ; ++i) {
                    const float4 x = raw4(i);
                    odd = look(x, odd);
                    big = max3(big, max3(fabsf(x.x), fabsf(x.y), fabsf(x.z)), fabsf(x.w));
                }
                // A row's queries have a power of two of their own, which no digits hang on, so that their largest is no more than 2: a score far below zero
                // would else be the difference of its parts' infinities.
                const int e = max(-126, min(60, 127 - (int)(__float_as_uint(big) >> 23)));
                up *= power2(e);
                factor = fminf(factor * power2(-e), 3.4e38f);
                const uint64_t up2 = pair(up, up);
                odd_queries = __any_sync(0xffffffffu, is_odd(odd));
#pragma unroll 1
                for (int part = 0; part < kPerQ / 4; ++part) {   // 16 elements: 8 columns of each part
                    uint32_t hi[8], mid[8], lo[8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float4 x = raw4(part * 4 + i);
                        const float2 front = unpair(mul2(pair(x.x, x.y), up2)), back = unpair(mul2(pair(x.z, x.w), up2));
                        split3(front.x, front.y, hi[2 * i], mid[2 * i], lo[2 * i]);
                        split3(back.x, back.y, hi[2 * i + 1], mid[2 * i + 1], lo[2 * i + 1]);
                    }
                    tmem_st_32x32b_x8(my_tmem + F::kQuery + part * 8, hi);
                    tmem_st_32x32b_x8(my_tmem + F::kQuery + DP / 2 + part * 8, mid);
                    tmem_st_32x32b_x8(my_tmem + F::kQuery + DP + part * 8, lo);
                }
            } else {
#pragma unroll
                for (int part = 0; part < kPerQ / 4; ++part) {   // 32 elements: 16 columns
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint4 r = raw(part * 4 + i);
                        const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) w[4 * i + k] = a.scale > 0.f ? u[k] : a.scale < 0.f ? u[k] ^ 0x80008000u : 0u;
                    }
                    tmem_st_32x32b_x16(my_tmem + F::kQuery + part * 16, w);
                }
            }
            tmem_st_wait();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&bar.q_full));
        }
        // All rows see all of a tile that lies between these.
        const uint32_t r_first = min(rt * kRows, n_rows - 1), r_last = min((rt + 1) * kRows, n_rows) - 1;
        const int32_t common_hi = key_bounds(a, first + per_head(r0 + r_first), length).hi, common_lo = key_bounds(a, first + per_head(r0 + max(r_last, r_first)), length).lo;
        // ... the tiles full_from .. full_to - 1
        const uint32_t full_from = sink_tiles + (uint32_t)max(0, (common_lo - span.lo + kKeys - 1) / kKeys);
        const uint32_t full_to = sink_tiles + (uint32_t)max(0, (min(span.hi, common_hi) - span.lo) / kKeys);
        float m = -INFINITY, l = 0.f;   // what weights are formed against; their sum, times 2^kBoost
        const uint32_t out_at = my_tmem + F::kProduct, columns = (dim + 15) / 16 * 16;   // the products write those; behind them lies what other kernels left
        // The output of the tiles since the last chunk's end is in tensor memory; that of those before in shared memory, against m_o
        float m_o = -INFINITY;
        bool o_any = false;
        // ... both together, times norm
        auto add_chunk = [&](bool chunk, float norm) {
            const float against = m == -INFINITY ? 0.f : m, f = exp2_approx(m_o - against) * norm;
#pragma unroll 1
            for (uint32_t col = 0; col < columns; col += 16) {
                uint32_t v[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = 0;
                if (chunk) {
                    tmem_ld_32x32b_x16(out_at + col, v);
                    tmem_ld_wait();
                }
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    float4& at = s_o[out_place(r, (col + i) / 4)];
                    float4 x = make_float4(__uint_as_float(v[i]) * norm, __uint_as_float(v[i + 1]) * norm, __uint_as_float(v[i + 2]) * norm, __uint_as_float(v[i + 3]) * norm);
                    if (o_any) {
                        const float4 y = at;
                        x = make_float4(fmaf(y.x, f, x.x), fmaf(y.y, f, x.y), fmaf(y.z, f, x.z), fmaf(y.w, f, x.w));
                    }
                    at = norm == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : x;   // (a row that sees nothing may hold what others' values left)
                }
            }
            m_o = m;
            o_any = true;
        };
        // Which of a tile's keys, from k0 on, this row sees
        auto seen_of = [&](int32_t k0, int32_t end) -> uint64_t {
            return below((int64_t)min(end, mine.hi) - k0) & ~(below((int64_t)mine.lo - k0) & ~below((int64_t)a.sinks - k0));
        };
        // A tile's scores, one by one, to `at`: where keys or queries are not finite
        auto scores_one_by_one = [&](uint32_t tile, uint32_t at) {
            const T* q = static_cast<const T*>(a.q) + (int64_t)b * a.q_batch + (int64_t)qi * a.q_token + (int64_t)(g * per_head.d + (row - qi * per_head.d)) * a.q_head;
            int32_t k0, end;
            tile_keys(tile, k0, end);
#pragma unroll 1
            for (uint32_t i = FEW ? warp * 16 : 0; i < (FEW ? warp * 16 + 16 : 64); ++i) {
                const int32_t key = k0 + (int32_t)i;
                float d = 0.f;
                if (key < end && (key < gap_from || key >= gap_to)) {
                    const T* k = static_cast<const T*>(a.k) + (int64_t)b * a.k_batch + (int64_t)g * a.k_head + (int64_t)key * a.k_token;
#pragma unroll 2
                    for (uint32_t c = 0; c < dim; c += kPer16<T>) {
                        float x[kPer16<T>], y[kPer16<T>];
                        load_elems<T, kPer16<T>>(q + c, x);
                        load_elems<T, kPer16<T>>(k + c, y);
#pragma unroll
                        for (int e = 0; e < kPer16<T>; ++e) d = fmaf(x[e] * up, y[e], d);
                    }
                }
                __syncwarp();
                tmem_st_32x32b_x1(at + i, __float_as_uint(d));
            }
            tmem_st_wait();
        };
        // What this row sees of values that are not finite, to its results
        auto add_odd_values = [&] {
            constexpr int kE = kPer16<T>, kBatch = 4;
            const T* const v_head = static_cast<const T*>(a.v) + (int64_t)b * a.v_batch + (int64_t)g * a.v_head;
            // (the loading warps may be at later tiles, and move the bounds: one lane reads them)
            const uint32_t from = __shfl_sync(0xffffffffu, *static_cast<volatile uint32_t*>(&s_odd_from[1]), 0);
            const uint32_t to = __shfl_sync(0xffffffffu, min(tiles, *static_cast<volatile uint32_t*>(&s_odd_to[1])), 0);
#pragma unroll 1
            for (uint32_t j = from; j < to; ++j) {
                if (RT == 2 && !sees(t0 + j)) continue;
                int32_t k0, end;
                tile_keys(t0 + j, k0, end);
                uint64_t seen = seen_of(k0, end);
                if (FEW) seen &= 0xFFFFull << (16 * warp);
                bool settled = true;   // nothing changes NaN
#pragma unroll 1
                for (uint32_t c = 0; c < dim; c += 4) {
                    const float4 x = s_o[out_place(r, c / 4)];
                    settled &= x.x != x.x && x.y != x.y && x.z != x.z && x.w != x.w;
                }
                if (__all_sync(0xffffffffu, settled)) break;
#pragma unroll 1
                for (uint32_t i = 0; i < 64; ++i) {
                    const bool me = seen >> i & 1u;
                    if (!__any_sync(0xffffffffu, me)) continue;
                    const T* v = v_head + (int64_t)(k0 + (int32_t)i) * a.v_token;
#pragma unroll 1
                    for (uint32_t c0 = 0; c0 < dim; c0 += kBatch * kE) {
                        float x[kBatch][kE];
#pragma unroll
                        for (int u = 0; u < kBatch; ++u) load_elems<T, kE>(v + (c0 + u * kE < dim ? c0 + u * kE : 0), x[u]);
#pragma unroll
                        for (int u = 0; u < kBatch; ++u)
#pragma unroll
                            for (int e = 0; e < kE; ++e) {
                                const uint32_t c = c0 + u * kE + e;
                                if (me && c < dim && !finite(x[u][e])) reinterpret_cast<float*>(&s_o[out_place(r, c / 4)])[c % 4] += x[u][e];
                            }
                    }
                }
            }
        };
        uint32_t n = 0;   // tiles so far
        // The last chunk's output, behind its last product
        auto end_chunk = [&]() -> bool {
            if (!wait_warp(smem_u32(&bar.done[(n - 1) & 1u]), ((n - 1) >> 1) & 1u, &s_abort)) return false;
            tc_fence_after_sync();
            add_chunk(true, 1.f);
            return true;
        };
        auto tile = [&](uint32_t j) -> bool {
            if (RT == 2 && !sees(t0 + j)) return true;
            if (F::kFp32 && n > 0 && first_row < n_rows) {   // while this tile's scores are formed
                if (!end_chunk()) return false;
            }
            if (!wait_warp(smem_u32(&bar.s_full[n & 1u]), (n >> 1) & 1u, &s_abort)) return false;
            tc_fence_after_sync();
            if (first_row >= n_rows) {   // a warp without rows: its weights are whatever lies there, and its output nobody's
                if (lane == 0) mbar_arrive(smem_u32(&bar.p_full[n & 1u]));
                ++n;
                return true;
            }
            const uint32_t at = my_tmem + F::kScores + n % F::kBufs * F::kScoreCols;
            float c = fmaxf(factor, 1.17549435e-38f);   // hidden scores, minus infinity, stay that
            if constexpr (F::kFp32) {
                if (__builtin_expect(__any_sync(0xffffffffu, odd_queries || j < *static_cast<volatile uint32_t*>(&s_odd_to[0])), 0)) {
                    // (not for rows whose sum is no number any more, and with it their result)
                    if ((odd_queries || __any_sync(0xffffffffu, j >= *static_cast<volatile uint32_t*>(&s_odd_from[0]))) && !__all_sync(0xffffffffu, l != l)) scores_one_by_one(t0 + j, at);
                }
            }
            constexpr int kGroups = FEW ? 1 : 2, kWide = FEW ? 16 : 32;
            uint32_t sc[kGroups][kWide];
            if constexpr (FEW) {
                tmem_ld_32x32b_x16(at + warp * 16, sc[0]);
            } else {
#pragma unroll
                for (int g = 0; g < 2; ++g) tmem_ld_32x32b_x32(at + g * 32, sc[g]);
            }
            tmem_ld_wait();
            if (t0 + j < full_from || t0 + j >= full_to) {
                int32_t k0, end;
                tile_keys(t0 + j, k0, end);
                const uint64_t seen = seen_of(k0, end);
#pragma unroll
                for (int g = 0; g < kGroups; ++g) {
                    const uint32_t bits = (uint32_t)(seen >> (FEW ? 16 * warp : 32 * g));
#pragma unroll
                    for (int i = 0; i < kWide; ++i)
                        if (!(bits >> i & 1u)) sc[g][i] = 0xFF800000u;
                }
            }
            float top;
            {
                float x = -INFINITY, y = -INFINITY;
#pragma unroll
                for (int g = 0; g < kGroups; ++g)
#pragma unroll
                    for (int i = 0; i < kWide; i += 4) {
                        x = max3(x, __uint_as_float(sc[g][i]), __uint_as_float(sc[g][i + 1]));
                        y = max3(y, __uint_as_float(sc[g][i + 2]), __uint_as_float(sc[g][i + 3]));
                    }
                top = fmaxf(x, y) * c;
            }
            top = ceilf(top);
            // The distance to the maximum is formed with one rounding, of itself.  Where a score's own is as large as that, its product is to be rounded as the
            // maximum's is, or the largest would lie that far from it.
            constexpr float kLarge = 4194304.f;
            auto round_products = [&] {
#pragma unroll
                for (int g = 0; g < kGroups; ++g)
#pragma unroll
                    for (int i = 0; i < kWide; ++i) sc[g][i] = __float_as_uint(__uint_as_float(sc[g][i]) * c);
                c = 1.f;
            };
            if constexpr (F::kFp32) {
                const float m_new = fmaxf(m, top);
                l *= m == -INFINITY ? 1.f : exp2_approx(m - m_new);
                m = m_new;
                if (__builtin_expect(fabsf(m) >= kLarge, 0)) round_products();
            } else {
                // A maximum that has grown by far: the output so far is brought in line, where there is one.
                if (m == -INFINITY) m = top;
                const bool grown = top > m + kSlack;
                if (__any_sync(0xffffffffu, grown || (fabsf(m) >= kLarge && m > -INFINITY))) {
                    const float m_new = grown ? top : m;
                    const float shrink = m == -INFINITY ? 1.f : exp2_approx(m - m_new);
                    if (n % F::kChunk != 0 && __any_sync(0xffffffffu, grown)) {
                        if (!wait_warp(smem_u32(&bar.done[(n - 1) & 1u]), ((n - 1) >> 1) & 1u, &s_abort)) return false;
                        tc_fence_after_sync();
#pragma unroll 1
                        for (uint32_t col = 0; col < columns; col += 16) {
                            uint32_t v[16];
                            tmem_ld_32x32b_x16(out_at + col, v);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * shrink);
                            tmem_st_32x32b_x16(out_at + col, v);
                        }
                        tmem_st_wait();
                    }
                    l *= shrink;
                    m = m_new;
                    if (__builtin_expect(fabsf(m) >= kLarge, 0)) round_products();
                }
            }
            const float boost = F::kFp32 ? 0.f : std::is_same<T, __half>::value ? kBoost : -kSlack - (float)log_keys;   // (fp32: in the values)
            const float more = boost - (m == -INFINITY ? 0.f : m);
            const uint64_t off = pair(more, more), cc = pair(c, c);
            uint64_t sum[2] = {0, 0};
            // Weights of 16 keys: 8 columns for each part.
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
#pragma unroll
                for (int part = 0; part < kWide / 16; ++part) {
                    const uint32_t to = at + (FEW ? warp : 2 * g + part) * 8;
                    uint32_t hi[8], mid[8], lo[8];
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        const float2 x = unpair(fma2(pair(__uint_as_float(sc[g][part * 16 + i]), __uint_as_float(sc[g][part * 16 + i + 1])), cc, off));
                        const float p = exp2_approx(x.x), q = exp2_approx(x.y);
                        sum[i / 2 & 1] = add2(sum[i / 2 & 1], pair(p, q));
                        if constexpr (F::kFp32) split3(p, q, hi[i / 2], mid[i / 2], lo[i / 2]);
                        else split2<T>(p, q, hi[i / 2], mid[i / 2]);
                    }
                    tmem_st_32x32b_x8(to, hi);
                    tmem_st_32x32b_x8(to + 32, mid);
                    if constexpr (F::kFp32) tmem_st_32x32b_x8(to + 64, lo);
                }
            }
            if constexpr (FEW) {   // the other warps' keys have no weight here
                const uint32_t none[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
                for (int i = 1; i < 4; ++i) {
#pragma unroll
                    for (int part = 0; part < (F::kFp32 ? 3 : 2); ++part) tmem_st_32x32b_x8(at + ((warp + i) & 3u) * 8 + part * 32, none);
                }
            }
            tmem_st_wait();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&bar.p_full[n & 1u]));
            const float2 sums = unpair(add2(sum[0], sum[1]));
            l = F::kFp32 ? fmaf(sums.x + sums.y, power2(-log_keys), l) : l + (sums.x + sums.y);
            ++n;
            return true;
        };
        for (uint32_t j = 0, ok = 1; ok && j < tiles;) {
            const uint32_t end = F::kFp32 ? tiles : min(tiles, j + F::kChunk);   // (16-bit types: one tile of rows, which sees all tiles)
            for (; ok && j < end; ++j) ok = tile(j);
            if (!F::kFp32 && ok && j < tiles && first_row < n_rows) ok = end_chunk();
        }
        const bool done = n > 0 && wait_warp(smem_u32(&bar.done[(n - 1) & 1u]), ((n - 1) >> 1) & 1u, &s_abort);
        tc_fence_after_sync();
        const float norm = FEW || shares > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l;
        add_chunk(done, norm);
        if (__builtin_expect(__any_sync(0xffffffffu, done && *static_cast<volatile uint32_t*>(&s_odd_to[1])), 0) && first_row < n_rows) add_odd_values();
        if (FEW || shares > 1) {
            s_m[r] = m;
            s_l[r] = l;
        } else {   // the warp's rows, whole lines at a time
            __syncwarp();
            constexpr uint32_t kE = kPer16<T>, kPerO = DP / kE;   // pieces of 16 bytes a row
            const uint32_t c = lane % kPerO * kE;
#pragma unroll 4
            for (uint32_t i = lane / kPerO; i < 32; i += 32 / kPerO) {
                if (warp_row + i >= n_rows || c >= dim) continue;
                float v[kE];
#pragma unroll
                for (uint32_t e = 0; e < kE; e += 4) {
                    const float4 x = s_o[out_place(warp_row + i, (c + e) / 4)];
                    v[e] = x.x; v[e + 1] = x.y; v[e + 2] = x.z; v[e + 3] = x.w;
                }
                store_elems<T, kE>(row_at(warp_row + i) + c, v);
            }
        }
    } else if (warp < F::kIssueAt) {
        // ---------------------------------------------------------------- keys and values into shared memory
        regs_down<F::kLoadRegs>();
        auto publish = [&](uint32_t job) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&s_full_bar[job % kSlots]));
        };
        for (uint32_t job = wg; job < jobs; job += RT) {
            if (job + F::kAhead * RT < jobs) copy(job + F::kAhead * RT);
            asm volatile("cp.async.commit_group;" ::: "memory");
            asm volatile("cp.async.wait_group %0;" ::"n"(F::kAhead) : "memory");
            if constexpr (F::kFp32) {   // in place, from what this thread has copied itself
                unsigned char* at = smem + job % kSlots * F::kTile;
                float4 buf[kPerThread];
                uint64_t odd = 0;
                const float down = power2(job & 1u ? -log_keys : 0);
                const uint64_t down2 = pair(down, down);
#pragma unroll
                for (int i = 0; i < kPerThread; ++i) {
                    const float4 x = *reinterpret_cast<const float4*>(at + i * 2048 + t * 16);
                    odd = look(x, odd);
                    const float2 front = unpair(mul2(pair(x.x, x.y), down2)), back = unpair(mul2(pair(x.z, x.w), down2));
                    buf[i] = make_float4(front.x, front.y, back.x, back.y);
                }
                sync_128(1 + wg);   // everybody has read
                if (is_odd(odd)) {
                    atomicMin(&s_odd_from[job & 1u], job / 2);
                    atomicMax(&s_odd_to[job & 1u], job / 2 + 1);
#pragma unroll
                    for (int i = 0; i < kPerThread; ++i) {
                        buf[i].x = finite(buf[i].x) ? buf[i].x : 0.f; buf[i].y = finite(buf[i].y) ? buf[i].y : 0.f;
                        buf[i].z = finite(buf[i].z) ? buf[i].z : 0.f; buf[i].w = finite(buf[i].w) ? buf[i].w : 0.f;
                    }
                }
#pragma unroll
                for (int i = 0; i < kPerThread; ++i) {
                    uint32_t hi[2], mid[2], lo[2];
                    split3(buf[i].x, buf[i].y, hi[0], mid[0], lo[0]);
                    split3(buf[i].z, buf[i].w, hi[1], mid[1], lo[1]);
                    unsigned char* to = at + place_of(i);
                    *reinterpret_cast<uint2*>(to) = make_uint2(hi[0], hi[1]);
                    *reinterpret_cast<uint2*>(to + F::kPart) = make_uint2(mid[0], mid[1]);
                    *reinterpret_cast<uint2*>(to + 2 * F::kPart) = make_uint2(lo[0], lo[1]);
                }
            }
            publish(job);
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    } else {
        // ---------------------------------------------------------------- the tensor core's instructions
        // A warp for the scores of each tile of rows, another for its products: what a tile costs such a warp - looking at barriers, issuing, committing -
        // is as long as the tensor core's work, and the two need not wait for one another.  All waits but the queries' are for the barriers of every other
        // tile, whose next phase cannot end before this one has been seen.
        regs_down<F::kIssueRegs>();
        const uint32_t rt = (warp - F::kIssueAt) % RT, role = (warp - F::kIssueAt) / RT;
        RowBars& bar = s_row[rt];
        const Seen sees = rows_see(rt);
        const uint32_t my_tmem = tmem + rt * 256u;
        auto wait_full = [&](uint32_t job) { return wait_warp(smem_u32(&s_full_bar[job % kSlots]), (job / kSlots) & 1u, &s_abort); };
        auto hand_back = [&](uint32_t job) {   // unread
            const bool ok = wait_full(job);
            if (ok && lane == 0) mbar_arrive(smem_u32(&s_empty_bar[job % kSlots]));
            return ok;
        };
        uint32_t n = 0;   // tiles that these rows see, so far
        // The products of parts, the small ones first: of fp32 (0, 2) (2, 0) (1, 1) (0, 1) (1, 0) (0, 0), of 16-bit types' weights (1, 0) (0, 0)
        constexpr int kTerms = F::kFp32 ? 6 : 1, kWeightTerms = F::kFp32 ? 6 : 2;
        auto left = [](int term) -> uint32_t { return F::kFp32 ? 0x021010u >> (4 * (5 - term)) & 0xFu : 0u; };
        auto right = [](int term) -> uint32_t { return F::kFp32 ? 0x201100u >> (4 * (5 - term)) & 0xFu : 0u; };
        auto weight = [&](int term) -> uint32_t { return F::kFp32 ? left(term) : 1u - term; };
        if (role == 0) {
            const uint32_t k_steps = (dim + 15) / 16, idesc = idesc_f16<T>(kKeys);
            bool ok = wait_warp(smem_u32(&bar.q_full), 0, &s_abort);
            for (uint32_t j = 0; ok && j < tiles; ++j) {
                if (!sees(t0 + j)) {
                    ok = hand_back(2 * j);
                    continue;
                }
                // S = Q K^T goes where the weights of the last tile, or of the one before, lie: its product has to be done
                if (n >= F::kBufs) ok = wait_warp(smem_u32(&bar.done[(n - F::kBufs) & 1u]), ((n - F::kBufs) >> 1) & 1u, &s_abort);
                ok = ok && wait_full(2 * j);
                if (!ok) break;
                tc_fence_after_sync();
                if (elect_one()) {
                    const uint32_t d = my_tmem + F::kScores + n % F::kBufs * F::kScoreCols;
                    const uint64_t keys = umma_desc_k_sw128(smem_at + 2 * j % kSlots * F::kTile);
                    auto issue = [&](uint32_t steps) {
#pragma unroll
                        for (int term = 0; term < kTerms; ++term) {
#pragma unroll
                            for (uint32_t s = 0; s < DP / 16; ++s) {
                                if (s >= steps) break;
                                const uint32_t at = right(term) * F::kPart + s / 4 * kPanel + s % 4 * 32;
                                umma_f16_ts(d, my_tmem + F::kQuery + left(term) * (DP / 2) + s * 8, keys + (at >> 4), idesc, term > 0 || s > 0);
                            }
                        }
                    };
                    if (k_steps == DP / 16) issue(DP / 16);
                    else issue(k_steps);
                    umma_commit(smem_u32(&bar.s_full[n & 1u]));
                    umma_commit(smem_u32(&s_empty_bar[2 * j % kSlots]));
                }
                __syncwarp();
                ++n;
            }
        } else if (role == 1) {
            uint32_t idescs[F::kPanels];
#pragma unroll
            for (int panel = 0; panel < F::kPanels; ++panel) idescs[panel] = idesc_f16<T>((min(dim - panel * 64u, 64u) + 15) / 16 * 16) | kIdescColumnMajorB;
            bool ok = true;
            for (uint32_t j = 0; ok && j < tiles; ++j) {
                if (!sees(t0 + j)) {
                    ok = hand_back(2 * j + 1);
                    continue;
                }
                ok = F::kFp32 ? wait_full(2 * j + 1) : wait_warp(smem_u32(&s_looked_bar[(2 * j + 1) % kSlots]), ((2 * j + 1) / kSlots) & 1u, &s_abort);
                ok = ok && wait_warp(smem_u32(&bar.p_full[n & 1u]), (n >> 1) & 1u, &s_abort);
                if (!ok) break;
                tc_fence_after_sync();
                if (elect_one()) {
                    const uint32_t p = my_tmem + F::kScores + n % F::kBufs * F::kScoreCols;
                    const uint64_t values = desc_rows(smem_at + (2 * j + 1) % kSlots * F::kTile);
                    const uint32_t go_on = n % F::kChunk != 0;
#pragma unroll
                    for (int panel = 0; panel < F::kPanels; ++panel) {
#pragma unroll
                        for (int term = 0; term < kWeightTerms; ++term) {
#pragma unroll
                            for (uint32_t s = 0; s < 4; ++s) {
                                const uint32_t at = right(term) * F::kPart + panel * kPanel + s * 2048;
                                umma_f16_ts(my_tmem + F::kProduct + panel * 64, p + weight(term) * 32 + s * 8, values + (at >> 4), idescs[panel], term > 0 || s > 0 ? 1u : go_on);
                            }
                        }
                    }
                    umma_commit(smem_u32(&bar.done[n & 1u]));
                    umma_commit(smem_u32(&s_empty_bar[(2 * j + 1) % kSlots]));
                }
                __syncwarp();
                ++n;
            }
        } else if constexpr (!F::kFp32) {
            // The two warps that are left look at the values, while weights are formed: where the loading warps did, single tokens behind eight caches took 62 us for 50.
            static_assert(RT == 1);
            for (uint32_t job = 1; job < jobs; job += 2) {
                if (!wait_full(job)) break;
                uint4* at = reinterpret_cast<uint4*>(smem + job % kSlots * F::kTile) + (role - 2) * 32 + lane;
                using T2 = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
                const uint32_t zero = 0;
                T2 odd[2] = {*reinterpret_cast<const T2*>(&zero), *reinterpret_cast<const T2*>(&zero)};
#pragma unroll
                for (int i = 0; i < F::kTile / 1024; ++i) {
                    const uint4 w = at[i * 64];
                    odd[0] = look(w.x, odd[0]); odd[1] = look(w.y, odd[1]); odd[0] = look(w.z, odd[0]); odd[1] = look(w.w, odd[1]);
                }
                const T2 all = __hadd2(odd[0], odd[1]);
                if (__builtin_expect(!(__low2float(all) == 0.f && __high2float(all) == 0.f), 0)) {
                    atomicMin(&s_odd_from[1], job / 2);
                    atomicMax(&s_odd_to[1], job / 2 + 1);
#pragma unroll 1
                    for (int i = 0; i < F::kTile / 1024; ++i) {
                        const uint4 w = at[i * 64];
                        at[i * 64] = make_uint4(only_finite<T>(w.x), only_finite<T>(w.y), only_finite<T>(w.z), only_finite<T>(w.w));
                    }
                    fence_proxy_async_smem();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&s_looked_bar[job % kSlots]));
            }
        }
    }

    if constexpr (FEW) {   // the four warps' parts into the first one's place
        __syncthreads();
        for (uint32_t i = tid; i < n_rows * (DP / 4); i += kThreads) {
            const uint32_t r = i / (DP / 4), c = i % (DP / 4);
            float mk[4], top = -INFINITY, total = 0.f;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < 4; ++w) top = fmaxf(top, mk[w] = s_m[w * 32 + r]);
#pragma unroll
            for (int w = 0; w < 4; ++w) add_part(v, total, s_o[out_place(w * 32 + r, c)], s_l[w * 32 + r], mk[w] == -INFINITY ? 0.f : exp2_approx(mk[w] - top));
            s_o[out_place(r, c)] = v;
            if (c == 0) {
                s_join[0][r] = top;
                s_join[FEW][r] = total;
            }
        }
    }
    if (FEW || shares > 1) {   // the CTAs' parts, four at a time on their way
        if (shares > 1) cluster_sync(); else __syncthreads();
        const float *from_m = FEW ? s_join[0] : s_m, *from_l = FEW ? s_join[FEW] : s_l;
        for (uint32_t i = share * kThreads + tid; i < n_rows * (DP / 4); i += shares * kThreads) {
            const uint32_t r = i / (DP / 4), c = i % (DP / 4), at_o = smem_u32(&s_o[out_place(r, c)]), at_m = smem_u32(from_m + r), at_l = smem_u32(from_l + r);
            if (c * 4 >= dim) continue;
            float top = -INFINITY, total = 0.f;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            for (uint32_t k0 = 0; k0 < shares; k0 += 4) {
                float mk[4], lk[4], most = top;
                float4 x[4];
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k) {
                    const bool in = k0 + k < shares;
                    mk[k] = in ? load_shared_cluster(map_to_rank(at_m, k0 + k)) : -INFINITY;
                    lk[k] = in ? load_shared_cluster(map_to_rank(at_l, k0 + k)) : 0.f;
                    x[k] = in ? load_shared_cluster4(map_to_rank(at_o, k0 + k)) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k) most = fmaxf(most, mk[k]);
                const float4 before = v;
                const float total_before = total, f = top == -INFINITY ? 0.f : exp2_approx(top - most);
                v = make_float4(0.f, 0.f, 0.f, 0.f);
                total = 0.f;
                add_part(v, total, before, total_before, f);
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k) add_part(v, total, x[k], lk[k], mk[k] == -INFINITY ? 0.f : exp2_approx(mk[k] - most));
                top = most;
            }
            const float norm = total == 0.f ? 0.f : 1.f / total;
            write_row(r, c * 4, make_float4(v.x * norm, v.y * norm, v.z * norm, v.w * norm));
        }
        if (shares > 1) cluster_sync();   // what the others read is read
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    if (warp == F::kIssueAt && s_abort) {   // what is in flight gets time to end before its columns are handed back
        const long long from = clock64();
        while (clock64() - from < 200000) {}
        if (lane == 0) report_error(dev_err, 7);
    }
    if (warp == F::kIssueAt) tmem_dealloc(tmem, F::kColumns);
}

template <typename T, int DP, int RT, bool FEW = false>
cudaError_t run(const AttentionArgs& a, int sm_count, uint32_t* dev_err, cudaStream_t s) {
    using F = Form<T, DP, RT>;
    static SmemOptIn memo;
    cudaError_t e = allow_smem(memo, attention_umma_kernel<T, DP, RT, FEW>, F::kSmem);
    if (e != cudaSuccess) return e;
    const uint64_t rows = (uint64_t)a.queries * (a.heads / a.kv_heads), tiles = (rows + RT * kRows - 1) / (RT * kRows);
    const uint64_t items = (uint64_t)a.batch * a.kv_heads * tiles;
    // Keys that a tile of rows sees at most.
    uint64_t keys = a.keys;
    if (a.left >= 0 && a.right >= 0) keys = std::min<uint64_t>(keys, (uint64_t)a.left + a.right + RT * kRows / (a.heads / a.kv_heads) + 1 + a.sinks);
    // As many shares as the SMs hold, by twos (clusters of three do not all find room: 48 items in thirds 42 us, in halves 29), of at least four tiles,
    // or two of fp32: joining them takes as long as those (256 tokens of 12 heads in bf16 in halves 12.0 us, whole 10.4; in fp32 in halves 13.0, whole
    // 16.3).
    constexpr uint32_t kShareTiles = sizeof(T) == 4 ? 2 : 4;
    uint32_t shares = 1;
    while (shares < kMostShares && items * shares * 2 <= (uint64_t)F::kCtas * sm_count && keys >= 2ull * shares * kShareTiles * kKeys) shares *= 2;
    if (rows > 0x7FFFFFFFull || items * shares > 0x7FFFFFFFull) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((uint32_t)(items * shares));
    cfg.blockDim = dim3(F::kThreads);
    cfg.dynamicSmemBytes = F::kSmem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = shares;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, attention_umma_kernel<T, DP, RT, FEW>, a, divisor((uint32_t)tiles), divisor(a.kv_heads), divisor(a.heads / a.kv_heads), dev_err);
}

template <typename T>
cudaError_t pick(const AttentionArgs& a, int sm_count, uint32_t* dev_err, cudaStream_t s) {
    const uint64_t rows = (uint64_t)a.queries * (a.heads / a.kv_heads);
    if (rows <= 32) return a.head_dim > 64 ? run<T, 128, 1, true>(a, sm_count, dev_err, s) : run<T, 64, 1, true>(a, sm_count, dev_err, s);
    if (a.head_dim > 64) return run<T, 128, 1>(a, sm_count, dev_err, s);
    // Two tiles of rows on one ring: fp32's keys and values are converted once for 256 rows, which pays where a window bounds them on both sides and there are CTAs for
    // all SMs (BERT-large's batch 98 us, 104 with CTAs of 128 rows, two on an SM; 8192 tokens with a window of 512 + 512 244 and 259).  Otherwise two CTAs overlap more
    // than that saves (ViT's batch 123 and 114 us, 16 x 512 tokens 139 and 127, one sequence of 256 18 and 13), as they do for 16-bit types, which are only copied (8192 tokens
    // in bf16 107 and 96, when there was such a form of them).
    if constexpr (sizeof(T) == 4) {
        const uint64_t items = (rows + 2 * kRows - 1) / (2 * kRows) * a.batch * a.kv_heads;
        if (a.left >= 0 && a.right >= 0 && rows > kRows && items >= (uint64_t)sm_count) return run<T, 64, 2>(a, sm_count, dev_err, s);
    }
    return run<T, 64, 1>(a, sm_count, dev_err, s);
}

}  // namespace

cudaError_t launch_attention_umma(const AttentionArgs& a, uint32_t dtype, int sm_count, uint32_t* dev_err, cudaStream_t s) {
    if (!a.batch || !a.queries || !a.heads) return cudaSuccess;
    return dtype == 0 ? pick<float>(a, sm_count, dev_err, s) : dtype == 1 ? pick<__half>(a, sm_count, dev_err, s) : pick<__nv_bfloat16>(a, sm_count, dev_err, s);
}

}  // namespace lutamm
