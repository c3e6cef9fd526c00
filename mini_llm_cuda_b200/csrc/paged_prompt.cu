// Paged attention of many rows of a sequence (prompts and chunks of prompts) on the 5th-generation tensor cores.
//
// A CTA takes a tile of 128 consecutive (token, query head) rows of one K/V head (two tiles with 4-bit pages) through the pages that any of them
// sees, 128 positions at a time:  S = Q K^T, P = exp2(S - m), O += P V. S (fp32) and O lie in tensor memory, P as bf16 over the columns of its
// S (heads of 64: beside it), so that it is the MMA's A operand from there. One warp brings K and V (TMA, a page at a time: 16 rows of 128-byte
// swizzled halves; with 4-bit pages four warps widen them), one issues the MMAs, and eight (four) warps take two threads (one) for a row: maximum,
// exponentials, sum. Two threads agree on the maximum by a barrier of their two warps, and exchange it only when one of them has a new one.
// Two CTAs (the two tiles) alternate on the tensor core: while one's products run, the other's exponentials are taken.
// O is rescaled only when a row's maximum has grown by more than 2^8 since the reference of its weights was set.
// A weight is rounded to bf16 for its product, half a step of 2^-8 relative to it, as the result is rounded after it; the sum takes it in fp32.
// Positions that no row of the CTA sees (behind the last one, between the first positions and the window) are zeros in V: 0 times what
// may lie there could be no number. A row whose result is not finite is done again from the formula (careful_row).
//
// What bounds it (bf16, heads of 128): not the tensor core (36 % of its cycles in the window below), the exponential's unit (32 %) or the issue slots (46 %), but the chain
// softmax -> P V -> next scores of each tile, 3500 cycles of which two tiles overlap; tensor memory holds no third tile and no second S. 8001
// tokens, 16 / 4 heads of 128: 262 us, 1000 TFLOP/s; in a window of 1024 104 us, 613 TFLOP/s, where a CTA's start and end (6 us of 26) tell.
#include <cstring>
#include <type_traits>

#include "paged_prompt.h"
#include "paged_row.cuh"
#include "tc_host.h"

namespace mlb {

namespace {

// Tiles of 128 rows of a CTA. One, and two CTAs on an SM, where TMA brings K and V: the CTAs alternate on the tensor core as the tiles of one would, and
// one's start and end lie under the other's steps. Two where warps widen 4-bit pages, which serves both.
template <typename KVT> constexpr int kPpTiles = sizeof(KVT) == 1 ? 2 : 1;
constexpr int kPpKeys = 128;                     // positions of a step
constexpr int kPpPages = kPpKeys / kKvBlock;
template <typename KVT> constexpr int kPpLoaders = sizeof(KVT) == 1 ? 4 : 1;                             // warps that bring K and V
// Threads of a row in the softmax. Two where TMA brings K and V: with one for all 128 positions a step's maximum and exponentials took 2200 cycles, twice
// the tile's products, and 8 such warps on an SM did not hide them. One with 4-bit pages, whose loaders and softmax share the issue slots that bound them.
template <typename KVT> constexpr int kPpHalves = sizeof(KVT) == 1 ? 1 : 2;
template <typename KVT> constexpr int kPpThreads = 128 * kPpHalves<KVT> * kPpTiles<KVT> + 32 * kPpLoaders<KVT> + 32;          // softmax warps, loaders, the issuer's
constexpr int kPpPoly = 8;                       // one pair of so many exponentials by polynomial (2: 4 % slower, 4: 2 %, none: none to 2 %)
constexpr float kPpLazy = 8.f;
constexpr uint32_t kPpSpin = 1u << 24;

__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, "
        "%22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
          "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr)
        : "memory");
}
// The registers of loads that tmem_ld_wait() has waited for: no use of them is moved before it
__device__ __forceinline__ void tmem_loaded(uint32_t (&r)[32]) {
    asm volatile(""
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                   "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]),
                   "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]),
                   "+r"(r[31]));
}
__device__ __forceinline__ void tmem_loaded(uint32_t (&r)[16]) {
    asm volatile(""
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                   "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]));
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
                 "r"(r[14]), "r"(r[15]), "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                   "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(addr)
                 : "memory");
}
// Largest of three; a NaN if one of them is
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float y;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
// 2^x of two numbers, x <= 128, without the exponential's unit: x = n + r with n the nearest whole number, 2^r by the cubic 1 + r (a + r (b + r c))
// whose largest relative error over -1/2 .. 1/2 is smallest (fitted by reweighted least squares: 1.0e-4, a twentieth of the half step of bf16
// that the weight is rounded by next), n added to the exponent. Below 2^-126: something below that, and exactly 0 from 2^-127 on.
__device__ __forceinline__ f32x2 ex2_poly(f32x2 x) {
    float a, d;
    unpack2(x, a, d);
    x = pack2(fmaxf(a, -127.f), fmaxf(d, -127.f));
    const float big = 12582912.f;                // 1.5 * 2^23: whole numbers are its low bits
    const f32x2 n = add2(x, pack2(big, big)), r = fma2(add2(n, pack2(-big, -big)), pack2(-1.f, -1.f), x);
    f32x2 y = fma2(pack2(0.05500893f, 0.05500893f), r, pack2(0.24221100f, 0.24221100f));
    y = fma2(y, r, pack2(0.69328290f, 0.69328290f));
    y = fma2(y, r, pack2(1.f, 1.f));
    float n0, n1;
    unpack2(n, n0, n1);
    unpack2(y, a, d);
    return pack2u(__float_as_uint(a) + (__float_as_uint(n0) << 23), __float_as_uint(d) + (__float_as_uint(n1) << 23));
}

// B operand whose N runs along the 128-byte rows (V: a row is a position, the dims are N): 64 dims a row, 128-byte swizzle, groups of
// eight positions 1024 bytes apart, the next 64 dims `next` bytes on.
__device__ __forceinline__ uint64_t umma_desc_rows_are_k(uint32_t smem_addr, uint32_t next) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr & 0x3FFFFu) >> 4);
    d |= (uint64_t)(next >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
// MMAs and commits are issued by a whole warp that elects a lane for each. Issued under `if (lane == 0)` an MMA took 100 to 215 cycles,
// whatever its size, since its operands have to be brought into uniform registers lane by lane there; this way 64, the tensor core's own
// for 128 x 128 x 16.
__device__ __forceinline__ void umma_ss(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p, one;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "elect.sync _|one, 0xffffffff;\n"
        "@one tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p, one;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "elect.sync _|one, 0xffffffff;\n"
        "@one tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
        "}\n" ::"r"(tmem_d),
        "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void commit_elected(uint32_t mbar) {
    asm volatile(
        "{\n"
        ".reg .pred one;\n"
        "elect.sync _|one, 0xffffffff;\n"
        "@one tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n"
        "}\n" ::"r"(mbar)
        : "memory");
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Heads of 64 dims leave room in tensor memory for weights beside the scores, so that the next step's scores are computed as soon as the
// softmax has this step's in its registers, under its exponentials. (A step of one tile took 3500 cycles, 1900 of them the softmax.)
template <typename KVT, int HD> constexpr bool kPpEarly = HD == 64 && kPpHalves<KVT> == 2;
template <int HD, int TILES, bool EARLY>
struct PromptSmem {
    static constexpr int stages = EARLY ? 2 : TILES;      // of K and V: with one, the other CTA of the SM fills the wait
    static constexpr uint32_t kQ = 128 * HD * 2, kKV = kPpKeys * HD * 2, kHalf = 128 * 128;      // bytes of a tile; of 64 dims of one
    static constexpr uint32_t q = 0, k = TILES * kQ, v = k + stages * kKV, bars = v + stages * kKV, total = bars + 256;
};
enum PromptBar { PB_KFULL = 0, PB_KEMPTY = 2, PB_VFULL = 4, PB_VEMPTY = 6, PB_Q = 8, PB_S = 9, PB_P = 11, PB_P2 = 13, PB_O = 15, PB_END = 17, PB_READ = 18, PB_COUNT = 19 };

template <typename KVT, int HD>
__global__ void __launch_bounds__(kPpThreads<KVT>, 3 - kPpTiles<KVT>)
    attn_prompt_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ AttnPagedParams p) {
    constexpr int TILES = kPpTiles<KVT>;
    constexpr bool EARLY = kPpEarly<KVT, HD>;
    using L = PromptSmem<HD, TILES, EARLY>;
    static_assert(!EARLY || TILES == 1, "columns of tensor memory");
    constexpr int NST = L::stages;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t sm0 = smem_u32(sm), bar0 = sm0 + L::bars;
    auto bar = [&](int i) { return bar0 + 8u * (uint32_t)i; };
    __shared__ uint32_t tmem_base;
    __shared__ int found[5];                     // sequence, tile in it, the sequence's first row, rows, positions
    constexpr int HALVES = kPpHalves<KVT>, COLS = kPpKeys / HALVES;       // positions of a step for a softmax thread
    __shared__ float shared_row[TILES][HALVES][128];      // of a row's two threads: maxima, then sums
    __shared__ unsigned odd_rows[TILES][HALVES][4];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr bool Q4 = sizeof(KVT) == 1;
    constexpr int kLoader = 4 * HALVES * TILES, kIssuer = kLoader + kPpLoaders<KVT>;

    if (warp == kIssuer) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)), "r"(256u * TILES) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        tc_fence_before();
    }
    if (warp == kLoader) {
        // which sequence's rows these are: those of sequences with more than kSplitRows, 128 TILES at a time, the last sequence and its later rows
        // (which see more) first; sequences are not ordered by length
        int want = (int)((gridDim.x - 1 - blockIdx.x) / (unsigned)p.c.kv_heads), at = -1;
        for (int b0 = 0; b0 < p.r.batch && at < 0; b0 += 32) {
            const int b = b0 + lane;
            int n = 0;
            PagedSeq s = {0, 0, 0};
            if (b < p.r.batch) {
                s = paged_seq(p.r, p.c.pt_stride, b, blockIdx.x == 0);
                const long long rows = (long long)s.n * p.group;
                n = rows > kSplitRows ? (int)((rows + 128 * TILES - 1) / (128 * TILES)) : 0;
            }
            int x = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            const unsigned has = __ballot_sync(0xffffffffu, want < x);
            if (has) {
                const int src = __ffs(has) - 1;
                at = b0 + src;
                want -= __shfl_sync(0xffffffffu, x - n, src);
                if (lane == src) { found[2] = s.r0; found[3] = s.n; found[4] = s.len; }
            } else {
                want -= __shfl_sync(0xffffffffu, x, 31);
            }
        }
        if (lane == 0) {
            found[0] = at;
            found[1] = want;
            for (int i = 0; i < PB_COUNT; ++i) {
                const bool filled = i == PB_KFULL || i == PB_KFULL + 1 || i == PB_VFULL || i == PB_VFULL + 1;
                mbar_init(bar(i), i == PB_Q ? 4 * HALVES * TILES : (i >= PB_P && i < PB_O) || i == PB_READ ? 4 * HALVES : Q4 && filled ? 128 : 1);
            }
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
    }
    __syncthreads();
    tc_fence_after();
    // Columns: S of each tile, then O of each, 128 apart, weights over their scores; or S, weights, O
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0), tmem_p = tmem + (EARLY ? 128 : 0), tmem_o = tmem + (EARLY ? 192 : TILES * 128);
    auto release = [&]() { asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256u * TILES)); };
    if (found[0] < 0) {                          // (uniform)
        if (warp == kIssuer) release();
        pdl_wait();
        return;
    }
    const int b = found[0], kvh = (int)((gridDim.x - 1 - blockIdx.x) % (unsigned)p.c.kv_heads), first = found[1] * 128 * TILES;
    const PagedSeq s = {found[2], found[3], found[4]};
    const int count = min(128 * TILES, s.n * p.group - first), tiles = TILES == 2 && count > 128 ? 2 : 1;
    const int pos0 = s.len - s.n, low = pos0 + per_group(p, first), high = pos0 + per_group(p, first + count - 1);
    const PagedSpan span = paged_span(p, low, high);
    const int steps = (span.count + kPpPages - 1) / kPpPages;
    auto wait = [&](int i, uint32_t parity) {
        if (mbar_wait_bounded(bar(i), parity, kPpSpin, 0)) return true;
        atomicExch(p.r.err, PG_WAIT);
        return false;
    };

    if (Q4 && warp >= kLoader && warp < kIssuer) {
        // a thread per position: its row of K, then of V, while the next step's codes are on their way
        const int i = tid - 32 * kLoader;
        constexpr int CW = HD / 8, SW = HD / 64;             // words of codes, of scales
        uint32_t kc[CW], ks[SW], vc[CW], vs[SW];
        auto load = [&](int j, bool is_k, uint32_t (&c)[CW], uint32_t (&sc)[SW]) {
            const int v = j * kPpPages + i / kKvBlock, pg = v < span.count ? span.page(v) : 0, key = pg * kKvBlock + i % kKvBlock;
            const bool use = v < span.count && key <= high && !(p.window > 0 && key <= low - p.window && key >= p.sinks);
#pragma unroll
            for (int e = 0; e < CW; ++e) c[e] = 0;
#pragma unroll
            for (int e = 0; e < SW; ++e) sc[e] = 0;
            if (!use) return;
            const size_t row = ((size_t)paged_page(p.c, p.r.err, b, pg, 0) * p.c.kv_heads + kvh) * kKvBlock + i % kKvBlock;
            const uint4* src = reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(is_k ? p.c.kpool : p.c.vpool) + row * (HD / 2));
            const uint32_t* ssrc = reinterpret_cast<const uint32_t*>((is_k ? p.c.kscale : p.c.vscale) + row * (HD / 16));
#pragma unroll
            for (int e = 0; e < CW / 4; ++e) {
                const uint4 x = __ldg(src + e);
                c[4 * e] = x.x; c[4 * e + 1] = x.y; c[4 * e + 2] = x.z; c[4 * e + 3] = x.w;
            }
#pragma unroll
            for (int e = 0; e < SW; ++e) sc[e] = __ldg(ssrc + e);
        };
        auto store = [&](uint32_t at, const uint32_t (&c)[CW], const uint32_t (&sc)[SW]) {
#pragma unroll
            for (int e = 0; e < CW; e += 4) {                // two scales at a time
                const uint32_t two = e4m3x2_to_f16(sc[e / 8] >> (e % 8 * 4));
                const float a = f16_lo(two) * kScaleUp, d = f16_hi(two) * kScaleUp;
                const uint32_t s0 = f32x2_to_bf16(a, a), s1 = f32x2_to_bf16(d, d);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int ch = e + u;
                    *reinterpret_cast<uint4*>(sm + at + ch / 8 * L::kHalf + i * 128 + ((ch % 8) ^ (i & 7)) * 16) = widen_codes(c[ch], u < 2 ? s0 : s1);
                }
            }
            fence_async_smem();
        };
        if (steps > 0) {
            load(0, true, kc, ks);
            load(0, false, vc, vs);
        }
        for (int j = 0; j < steps; ++j) {
            const int st = j % NST;
            const uint32_t ph = (uint32_t)(j / NST) & 1u;
            if (!wait(PB_KEMPTY + st, ph ^ 1u)) break;
            store(L::k + st * L::kKV, kc, ks);
            mbar_arrive(bar(PB_KFULL + st));
            if (j + 1 < steps) load(j + 1, true, kc, ks);
            if (!wait(PB_VEMPTY + st, ph ^ 1u)) break;
            store(L::v + st * L::kKV, vc, vs);
            mbar_arrive(bar(PB_VFULL + st));
            if (j + 1 < steps) load(j + 1, false, vc, vs);
        }
    } else if (!Q4 && warp == kLoader) {
        bool good = true;
        int filled[2] = {0, 0};                  // steps whose K, V are on their way or there
        for (int j = 0; j < steps && good; ++j) {
            const int st = j % NST;
            const uint32_t ph = (uint32_t)(j / NST) & 1u;
            const int v = j * kPpPages + (lane & 7), pg = v < span.count ? span.page(v) : 0;
            const bool held = lane < kPpPages && v < span.count;
            const int row0 = held ? (int)(((long long)paged_page(p.c, p.r.err, b, pg, 0) * p.c.kv_heads + kvh) * kKvBlock) : 0;
            const int key0 = pg * kKvBlock;
            // a page with positions that no row sees is copied by the warp, with zeros in their place
            const bool partly = key0 + kKvBlock - 1 > high || (p.window > 0 && key0 <= low - p.window && key0 + kKvBlock > p.sinks);
            const unsigned all = __ballot_sync(0xffffffffu, held), by_hand = __ballot_sync(0xffffffffu, lane < kPpPages && (!held || partly));
            good = __all_sync(0xffffffffu, wait(PB_KEMPTY + st, ph ^ 1u));
            if (!good) break;
            if (lane == 0) mbar_expect_tx(bar(PB_KFULL + st), (uint32_t)__popc(all) * kKvBlock * HD * 2);
            __syncwarp();
            if (held) {
#pragma unroll
                for (int h = 0; h < HD / 64; ++h)
                    tma_load_2d(sm0 + L::k + st * L::kKV + h * L::kHalf + lane * 2048, &tmK, h * 64, row0, bar(PB_KFULL + st));
            }
            filled[0] = j + 1;
            good = __all_sync(0xffffffffu, wait(PB_VEMPTY + st, ph ^ 1u));
            if (!good) break;
            for (unsigned left = by_hand; left; left &= left - 1) {
                const int i = __ffs(left) - 1, k0 = __shfl_sync(0xffffffffu, key0, i), r0 = __shfl_sync(0xffffffffu, row0, i);
                const bool here = (all >> i) & 1u;
                for (int e = lane; e < kKvBlock * HD / 8; e += 32) {
                    const int row = e / (HD / 8), ch = e % (HD / 8), key = k0 + row, at = i * kKvBlock + row;
                    uint4 x = make_uint4(0, 0, 0, 0);
                    if (here && key <= high && !(p.window > 0 && key <= low - p.window && key >= p.sinks))
                        x = __ldg(reinterpret_cast<const uint4*>(static_cast<const bf16_t*>(p.c.vpool) + (size_t)(r0 + row) * HD) + ch);
                    *reinterpret_cast<uint4*>(sm + L::v + st * L::kKV + ch / 8 * L::kHalf + at * 128 + ((ch % 8) ^ (at & 7)) * 16) = x;
                }
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_expect_tx(bar(PB_VFULL + st), (uint32_t)(kPpPages - __popc(by_hand)) * kKvBlock * HD * 2);
            __syncwarp();
            if (held && !partly) {
#pragma unroll
                for (int h = 0; h < HD / 64; ++h)
                    tma_load_2d(sm0 + L::v + st * L::kKV + h * L::kHalf + lane * 2048, &tmV, h * 64, row0, bar(PB_VFULL + st));
            }
            filled[1] = j + 1;
        }
        if (!good) {                             // no copy outlives the CTA
            for (int i = 0; i < 2; ++i)
                for (int j = max(0, filled[i] - NST); j < filled[i]; ++j) wait((i ? PB_VFULL : PB_KFULL) + j % NST, (uint32_t)(j / NST) & 1u);
        }
    } else if (warp == kIssuer) {
        if (steps > 0) {
            const uint32_t is = umma_idesc_bf16(128, kPpKeys), io = umma_idesc_bf16(128, HD) | (1u << 16);      // bit 16: N runs along B's rows
            auto scores = [&](int t, int j) {
#pragma unroll
                for (int ks = 0; ks < HD / 16; ++ks) {
                    const uint32_t off = (uint32_t)(ks / 4) * L::kHalf + (uint32_t)(ks % 4) * 32;
                    umma_ss(tmem + t * 128, umma_desc_sw128(sm0 + L::q + t * L::kQ + off), umma_desc_sw128(sm0 + L::k + j % NST * L::kKV + off), is, ks > 0);
                }
                commit_elected(bar(PB_S + t));
            };
            auto all_wait = [&](int i, uint32_t parity) { return __all_sync(0xffffffffu, wait(i, parity)) != 0; };
            bool good = all_wait(PB_Q, 0) && all_wait(PB_KFULL, 0);
            tc_fence_after();
            if (good) {
                for (int t = 0; t < tiles; ++t) scores(t, 0);
                commit_elected(bar(PB_KEMPTY));
            }
            for (int j = 0; j < steps && good; ++j) {
                const uint32_t ph = (uint32_t)(j / NST) & 1u;
                if (EARLY && j + 1 < steps) {
                    good = all_wait(PB_READ, (uint32_t)j & 1u) && all_wait(PB_KFULL + (j + 1) % NST, (uint32_t)((j + 1) / NST) & 1u);
                    if (!good) break;
                    tc_fence_after();
                    scores(0, j + 1);
                    commit_elected(bar(PB_KEMPTY + (j + 1) % NST));
                }
                for (int t = 0; t < tiles && good; ++t) {
                    good = all_wait(PB_P + t, (uint32_t)j & 1u) && (t > 0 || all_wait(PB_VFULL + j % NST, ph));
                    if (!good) break;
                    tc_fence_after();
#pragma unroll
                    for (int i = 0; i < kPpKeys / 16; ++i) {
                        // weights lie where the scores of their thread were; those of each thread's first positions come first
                        const int ks = HALVES == 2 ? (i & 1) + (i & 2) * 2 + (i & 4) / 2 : i;
                        if (i == kPpKeys / 32) {
                            good = all_wait(PB_P2 + t, (uint32_t)j & 1u);
                            if (!good) break;
                            tc_fence_after();
                        }
                        umma_ts(tmem_o + t * 128, tmem_p + t * 128 + (HALVES == 2 && !EARLY ? ks / 4 * 64 + ks % 4 * 8 : ks * 8), umma_desc_rows_are_k(sm0 + L::v + j % NST * L::kKV + ks * 2048, L::kHalf), io,
                                     j > 0 || i > 0);
                    }
                    if (!good) break;
                    if (t == tiles - 1) commit_elected(bar(PB_VEMPTY + j % NST));
                    if (j + 1 < steps) {
                        if (EARLY) continue;
                        if (t == 0) {
                            good = all_wait(PB_KFULL + (j + 1) % NST, (uint32_t)((j + 1) / NST) & 1u);
                            if (!good) break;
                            tc_fence_after();
                        }
                        scores(t, j + 1);
                        if (t == tiles - 1) commit_elected(bar(PB_KEMPTY + (j + 1) % NST));
                    } else {
                        commit_elected(bar(PB_O + t));
                    }
                }
            }
            if (!good) {                         // nor does a product
                commit_elected(bar(PB_END));
                all_wait(PB_END, 0);
            }
        }
    } else {
        // The warps of a row's two threads, four apart, share its 32 lanes of tensor memory.
        const int t = warp / (4 * HALVES), half = HALVES == 2 ? warp / 4 & 1 : 0, r = tid & 127, i = t * 128 + r;      // this thread's row of the CTA's
        const bool in = i < count;
        const int rr = first + (in ? i : 0), tok = per_group(p, rr), row = s.r0 + tok, h = kvh * p.group + rr - tok * p.group;
        const int pos = in ? pos0 + tok : high;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;            // the warp's 32 lanes of tensor memory
        const int pair = 1 + t * 4 + (warp & 3);                      // named barrier of the two warps of these rows
        auto pair_sync = [&]() {
            if constexpr (HALVES == 2) asm volatile("bar.sync %0, 64;" ::"r"(pair) : "memory");
            else __syncwarp();
        };
        auto pair_any = [&](bool x) {
            if constexpr (HALVES == 1) return __any_sync(0xffffffffu, x) != 0;
            uint32_t y;
            asm volatile(
                "{\n"
                ".reg .pred a, b;\n"
                "setp.ne.u32 a, %1, 0;\n"
                "bar.red.or.pred b, %2, 64, a;\n"
                "selp.u32 %0, 1, 0, b;\n"
                "}\n"
                : "=r"(y)
                : "r"((uint32_t)x), "r"(pair)
                : "memory");
            return y != 0;
        };
        // The tile's rows lie in memory by (token, head); a warp takes 16 or 32 of them, and CH lanes the 16-byte pieces of one, so that it reads and writes
        // whole rows: `piece(k)` is the k-th of a lane. (A row per thread: 4 us for the queries and 3 for the results.)
        constexpr int CH = HD / 8, NP = 32 / HALVES * CH / 32;
        struct Piece { int r, c; bool in; long long row, col; };
        auto piece = [&](int k) {
            Piece x;
            x.r = (warp & 3) * 32 + half * (32 / HALVES) + k * (32 / CH) + lane / CH;
            x.c = lane % CH;
            x.in = t * 128 + x.r < count;
            const int a = first + (x.in ? t * 128 + x.r : 0), token = per_group(p, a);
            x.row = s.r0 + token;
            x.col = (long long)(kvh * p.group + a - token * p.group) * HD + x.c * 8;
            return x;
        };
        auto staged = [&](int rl, int ch) { return reinterpret_cast<uint4*>(sm + L::q + t * L::kQ + ch / 8 * L::kHalf + rl * 128 + ((ch % 8) ^ (rl & 7)) * 16); };
        // queries, K-major with the swizzle that the MMA expects; a negative scale turns their sign
        const float scale = p.scale * p.c.k_scale * (Q4 ? kCodeScale : 1.f) * 1.4426950408889634f;
        {
            const bf16_t* q = static_cast<const bf16_t*>(p.q);
            const bool vec = ((reinterpret_cast<uintptr_t>(q) | (uint64_t)p.q_stride * 2) & 15) == 0;
            const uint32_t turn = scale < 0.f ? 0x80008000u : 0u;
            constexpr int NQ = NP < 8 ? NP : 8;                  // loads on their way at once
            for (int k0 = 0; k0 < NP; k0 += NQ) {
            uint4 x[NQ];
#pragma unroll
            for (int k = 0; k < NQ; ++k) {
                const Piece y = piece(k0 + k);
                const bf16_t* src = q + y.row * p.q_stride + y.col;
                x[k] = make_uint4(0, 0, 0, 0);
                if (y.in && vec) x[k] = __ldg(reinterpret_cast<const uint4*>(src));
                if (y.in && !vec) {
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = (uint32_t)__bfloat16_as_ushort(src[2 * e]) | (uint32_t)__bfloat16_as_ushort(src[2 * e + 1]) << 16;
                    x[k] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
#pragma unroll
            for (int k = 0; k < NQ; ++k) {
                uint4 v = x[k];
                v.x ^= turn; v.y ^= turn; v.z ^= turn; v.w ^= turn;
                if (Q4)                                          // the order of dims in K
                    v = make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.y, v.w, 0x7632));
                const Piece y = piece(k0 + k);
                *staged(y.r, y.c) = y.in ? v : make_uint4(0, 0, 0, 0);
            }
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(PB_Q));
        }
        const float c = fabsf(scale);
        float m = -INFINITY, l = 0.f;
        bool good = true;                        // (a warp whose wait ran out goes on without waiting: its partner's barriers need it)
        if (t < tiles) {
            // pages all of whose positions all of the warp's rows see: from inner0 on (first positions aside), before inner1
            const int wlow = __reduce_min_sync(0xffffffffu, pos), whigh = __reduce_max_sync(0xffffffffu, pos);
            const int inner0 = p.window > 0 ? span.sink_pages + max(0, (whigh - p.window + kKvBlock) / kKvBlock - span.first) : 0;
            const int inner1 = span.sink_pages + (wlow + 1) / kKvBlock - span.first;
            const uint32_t sc = tmem + lanes + t * 128 + half * COLS;
            // Scores: two threads of a row hold theirs in registers, one reads them twice, for the maximum and for the weights.
            constexpr int NG = COLS / 32;
            uint32_t x[2][32];
            for (int j = 0; j < steps; ++j) {
                good = good && __all_sync(0xffffffffu, wait(PB_S + t, (uint32_t)j & 1u));
                tc_fence_after();
                tmem_ld32(sc, x[0]);
                if (HALVES == 2) tmem_ld32(sc + 32, x[1]);
                const int v0 = j * kPpPages + half * (kPpPages / 2);
                const bool edge = v0 < inner0 || v0 + kPpPages / HALVES > inner1;      // positions that some row of the warp does not see
                // 32 positions from 32 g on: those that the row does not see to -inf
                auto hide = [&](uint32_t (&y)[32], int g) {
                    auto below = [](int n) { return (1u << min(max(n, 0), kKvBlock)) - 1u; };
                    uint32_t seen = 0;
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int v = v0 + 2 * g + u;
                        if (v < span.count) {
                            const int k0 = span.page(v) * kKvBlock, lo = p.window > 0 ? max(0, pos - p.window + 1) : 0;
                            seen |= (below(pos + 1 - k0) & (~below(lo - k0) | below(p.sinks - k0))) << (u * kKvBlock);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (!(seen >> e & 1u)) y[e] = 0xff800000u;
                };
                auto arrived = [&](int g) {                      // scores of group g are in x[g & 1], and the next ones on their way
                    if (HALVES == 1 || g == 0) tmem_ld_wait();
                    if (HALVES == 2 && g == 0) tmem_loaded(x[1]);
                    if (HALVES == 1 || g == 0) tmem_loaded(x[g & 1]);
                    if (HALVES == 1 && g + 1 < NG) tmem_ld32(sc + 32 * (g + 1), x[(g + 1) & 1]);
                    if (edge) hide(x[g & 1], g);
                };
                if constexpr (EARLY) {                           // (both halves of the scores are waited for together)
                    arrived(0);
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(PB_READ));
                }
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    if (!EARLY || g > 0) arrived(g);
#pragma unroll
                    for (int u = 0; u < 32; u += 2)
                        top[u / 2 & 3] = max3_nan(top[u / 2 & 3], __uint_as_float(x[g & 1][u]), __uint_as_float(x[g & 1][u + 1]));
                }
                float mx = max3_nan(max3_nan(top[0], top[1], top[2]), top[3], -INFINITY) * c;
                // the products with the step before's weights are done: O and the weights' columns are this step's
                if (EARLY && j > 0) {
                    good = good && __all_sync(0xffffffffu, wait(PB_VEMPTY + (j - 1) % NST, (uint32_t)((j - 1) / NST) & 1u));
                    tc_fence_after();
                }
                // (a score that is no number makes the maximum, and so the row, none)
                if (pair_any(!(mx <= m + kPpLazy))) {
                    if constexpr (HALVES == 2) {
                        shared_row[t][half][r] = mx;
                        pair_sync();
                        mx = max3_nan(mx, shared_row[t][half ^ 1][r], -INFINITY);
                    }
                    const bool moved = !(mx <= m + kPpLazy);
                    const float f = moved ? ex2(m - mx) : 1.f;
                    if (moved) m = mx;
                    l *= f;
                    if (j > 0) {
#pragma unroll 1
                        for (int e = half * (HD / 16 / HALVES); e < (half + 1) * (HD / 16 / HALVES); ++e) {
                            uint32_t o[16];
                            const uint32_t at = tmem_o + lanes + t * 128 + e * 16;
                            tmem_ld16(at, o);
                            tmem_ld_wait();
                            tmem_loaded(o);
#pragma unroll
                            for (int u = 0; u < 16; ++u) o[u] = __float_as_uint(__uint_as_float(o[u]) * f);
                            tmem_st16(at, o);
                        }
                    }
                }
                const float ref = m == -INFINITY ? 0.f : m;
                const f32x2 cc = pack2(c, c), rr2 = pack2(-ref, -ref);
                f32x2 sum[2] = {0ull, 0ull};
                if (HALVES == 1) tmem_ld32(sc, x[0]);
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    if (HALVES == 1) arrived(g);
                    // weights of 32 positions, some by polynomial: the exponential's unit takes 16 a cycle
                    uint32_t w[16];
#pragma unroll
                    for (int u = 0; u < 16; ++u) {
                        f32x2 y = fma2(pack2u(x[g & 1][2 * u], x[g & 1][2 * u + 1]), cc, rr2);
                        float a, d;
                        if (u % kPpPoly == kPpPoly - 1) {
                            y = ex2_poly(y);
                            unpack2(y, a, d);
                        } else {
                            unpack2(y, a, d);
                            a = ex2(a);
                            d = ex2(d);
                            y = pack2(a, d);
                        }
                        sum[u & 1] = add2(sum[u & 1], y);
                        w[u] = f32x2_to_bf16(a, d);
                    }
                    tmem_st16(EARLY ? tmem_p + lanes + half * 32 + 16 * g : sc + 16 * g, w);      // (over scores that have been read)
                    if ((g + 1) % (NG / 2) == 0) {               // half of the positions: their products can begin
                        tmem_st_wait();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(bar((g + 1 == NG / 2 ? PB_P : PB_P2) + t));
                    }
                }
                float sa, sb, sd, se;
                unpack2(sum[0], sa, sb);
                unpack2(sum[1], sd, se);
                l += (sa + sb) + (sd + se);
            }
            // results
            if (steps > 0) {
                good = good && __all_sync(0xffffffffu, wait(PB_O + t, 0));
                tc_fence_after();
            }
            if constexpr (HALVES == 2) {
                pair_sync();                                     // the maxima have been read
                shared_row[t][half][r] = l;
                pair_sync();
                l = shared_row[t][0][r] + shared_row[t][1][r];   // the same sum in both threads
            }
            const float inv = pos < 0 ? 0.f : p.c.v_scale * (Q4 ? kCodeScale : 1.f) / l;
            bool odd = false;
            if (good) {
#pragma unroll 1
                for (int e = half * (HD / 32 / HALVES); e < (half + 1) * (HD / 32 / HALVES); ++e) {
                    uint32_t o[32];
                    if (steps > 0) {
                        tmem_ld32(tmem_o + lanes + t * 128 + e * 32, o);
                        tmem_ld_wait();
                        tmem_loaded(o);
                    }
                    float y[32];
#pragma unroll
                    for (int u = 0; u < 32; ++u) {
                        const int from = !Q4 ? u : u / 8 * 8 + (u % 8 < 4 ? u % 8 * 2 : u % 8 * 2 - 7);      // the order of dims in V
                        y[u] = pos < 0 ? 0.f : __uint_as_float(o[from]) * inv;
                        odd |= !(fabsf(y[u]) <= 3.4e38f);
                    }
                    if (p.gate && in && pos >= 0) {
                        const float* gp = p.gate + (size_t)row * p.heads * HD + (size_t)h * HD + e * 32;
#pragma unroll
                        for (int u = 0; u < 32; ++u) y[u] *= gp[u];
                    }
#pragma unroll
                    for (int u = 0; u < 32; u += 8)              // where the queries were
                        *staged(r, e * 4 + u / 8) = make_uint4(f32x2_to_bf16(y[u], y[u + 1]), f32x2_to_bf16(y[u + 2], y[u + 3]),
                                                               f32x2_to_bf16(y[u + 4], y[u + 5]), f32x2_to_bf16(y[u + 6], y[u + 7]));
                }
            }
            pair_sync();
            if (good) {
                bf16_t* out = static_cast<bf16_t*>(p.out);
                const bool vec = ((reinterpret_cast<uintptr_t>(out) | (uint64_t)p.out_stride * 2) & 15) == 0;
#pragma unroll
                for (int k = 0; k < NP; ++k) {
                    const Piece y = piece(k);
                    if (!y.in) continue;
                    const uint4 v = *staged(y.r, y.c);
                    bf16_t* dst = out + y.row * p.out_stride + y.col;
                    if (vec) {
                        *reinterpret_cast<uint4*>(dst) = v;
                    } else {
                        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            dst[2 * e] = __ushort_as_bfloat16((unsigned short)(w[e] & 0xffffu));
                            dst[2 * e + 1] = __ushort_as_bfloat16((unsigned short)(w[e] >> 16));
                        }
                    }
                }
            }
            const unsigned mine = __ballot_sync(0xffffffffu, odd && in && good);
            if (lane == 0) odd_rows[t][half][warp & 3] = mine;
            pair_sync();                                         // (what either warp has written is written)
            // the pair's warps in turn
            unsigned again = (odd_rows[t][0][warp & 3] | odd_rows[t][HALVES - 1][warp & 3]) & (HALVES == 1 ? 0xffffffffu : half ? 0xaaaaaaaau : 0x55555555u);
            for (; again; again &= again - 1) {
                const int src = __ffs(again) - 1;
                careful_row<KVT, bf16_t, HD>(p, b, __shfl_sync(0xffffffffu, pos, src), __shfl_sync(0xffffffffu, row, src), __shfl_sync(0xffffffffu, h, src));
            }
        }
        tc_fence_before();
    }
    __syncwarp();
    __syncthreads();
    if (warp == kIssuer) {
        tc_fence_after();
        release();
    }
    pdl_wait();                                  // nothing here needs the kernels before, but the next one in the stream may, and it waits for this one alone
}

template <typename KVT, int HD>
cudaError_t launch(const AttnPagedParams& p, const PromptMaps& maps, cudaStream_t st) {
    const size_t smem = PromptSmem<HD, kPpTiles<KVT>, kPpEarly<KVT, HD>>::total + 1024;
    cudaError_t e = cudaFuncSetAttribute(attn_prompt_kernel<KVT, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    const long long tiles = (long long)p.r.rows * p.group / (128 * kPpTiles<KVT>) + p.r.batch;
    // It starts while the kernels of the short sequences, which it shares nothing with, are at work.
    return launch_after(attn_prompt_kernel<KVT, HD>, dim3((unsigned)(tiles * p.c.kv_heads)), kPpThreads<KVT>, smem, st, maps.k, maps.v, p);
}

}  // namespace

cudaError_t attn_prompt_maps(const AttnPagedParams& p, int dtype, int head_dim, PromptMaps* maps) {
    std::memset(maps, 0, sizeof *maps);
    if (dtype != MLB_DT_BF16) return cudaSuccess;
    static const EncodeTiledFn enc = get_encode_tiled();
    if (!enc) return cudaErrorNotSupported;
    const uint64_t rows = (uint64_t)p.c.num_pages * p.c.kv_heads * kKvBlock;
    if (make_bf16_map(enc, &maps->k, p.c.kpool, rows, head_dim, kKvBlock) || make_bf16_map(enc, &maps->v, p.c.vpool, rows, head_dim, kKvBlock)) return cudaErrorInvalidValue;
    return cudaSuccess;
}

cudaError_t attn_prompt_launch(const AttnPagedParams& p, int dtype, int head_dim, const PromptMaps& maps, cudaStream_t st) {
    if (dtype == MLB_DT_FP4_E2M1) return head_dim == 64 ? launch<fp4_t, 64>(p, maps, st) : launch<fp4_t, 128>(p, maps, st);
    return head_dim == 64 ? launch<bf16_t, 64>(p, maps, st) : launch<bf16_t, 128>(p, maps, st);
}

}  // namespace mlb
