// What the kernels of the paged attention share: a row of it straight from the formula, and the place of a result.
#pragma once
#include "paged.cuh"

namespace mlb {

// (results under 2^-126 are 0: without that, three more instructions)
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 4-bit pages: eight codes (dims 0 .. 7) -> four bf16 pairs (0, 4), (1, 5), (2, 6), (3, 7) of code * scale / 256. Exponent and mantissa of
// a code are put at the low end of a bf16's exponent, which makes it code * 2^-126 exactly (0.5 as a subnormal), and multiplied by `s`, the
// block's scale * 2^118 (once for each of a pair). In that order a pair takes two shifts, two logic instructions and a product. (The conversion instruction
// runs at a quarter of the rate of these and gives halves.)
__device__ __forceinline__ uint4 widen_codes(uint32_t w, uint32_t s) {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t sign = i < 3 ? w << (12 - 4 * i) : w, rest = i < 2 ? w << (6 - 4 * i) : w >> (4 * i - 6);
        const uint32_t raw = (sign & 0x80008000u) | (rest & 0x01c001c0u);
        asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r[i]) : "r"(raw), "r"(s));
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}
constexpr float kScaleUp = 3.3230699894622897e35f;      // 2^118
constexpr float kCodeScale = 256.f;            // what those values lack

// ---- one row, one head, by one warp, straight from the formula --------------------------------------------------------
// A product with a probability that is not of the row's own positions does not happen here, so infinities and NaN outside of them cannot
// reach the row, and an infinite score or value gives what the formula gives. The matrix-core kernels redo a row here whose result is
// not finite: there a probability of 0 times an infinity, or a piece of an infinite number, is a NaN. Two pages at a time, a lane for each position's score,
// then the lanes for the dims of V; it ends where nothing can be a number any more. A row that sees
// 20000 positions, heads of 128, bf16: 2.8 ms where one of its values is infinite, 35 us for the call where a key near the start is NaN (a position at a
// time and to the end: 10 ms for either); a prompt of 2000, 16 heads: 5.7 ms and 0.2 (34).
template <typename KVT, typename RT, int HD>
static __device__ __noinline__ void careful_row(const AttnPagedParams& p, int b, int pos, int row, int h) {
    constexpr int E = HD / 32;                   // dims of a lane
    constexpr bool Q4 = sizeof(KVT) == 1;
    const int lane = threadIdx.x & 31, kvh = h / p.group;
    const RT* qp = static_cast<const RT*>(p.q) + (size_t)row * p.q_stride + (size_t)h * HD;
    float o[E], top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
    const PagedSpan span = paged_span(p, pos, pos);
    const float scale = p.scale * p.c.k_scale;
    bool any = false;
    for (int v = 0; v < span.count; v += 2) {
        const int mine = v + lane / kKvBlock;    // this lane's page of the two
        int id = 0;
        bool sees = false;
        if (mine < span.count) {
            const int pg = span.page(mine);
            id = paged_page(p.c, p.r.err, b, pg, 0);
            sees = paged_sees(p, pos, pg * kKvBlock + lane % kKvBlock);
        }
        const unsigned seen = __ballot_sync(0xffffffffu, sees);
        any |= seen != 0;
        float s = -INFINITY;
        if (sees) {
            const size_t at = ((size_t)id * p.c.kv_heads + kvh) * kKvBlock + lane % kKvBlock;
            s = 0.f;
#pragma unroll 8
            for (int d = 0; d < HD; d += 8) {
                float x[8];
                if constexpr (Q4) {
                    const uint32_t codes = reinterpret_cast<const uint32_t*>(static_cast<const unsigned char*>(p.c.kpool) + at * (HD / 2))[d / 8];
                    const float one = e4m3_to_f32(p.c.kscale[at * (HD / 16) + d / 16]);
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = e2m1_value(codes >> (4 * e)) * one;
                } else {
                    const KVT* src = static_cast<const KVT*>(p.c.kpool) + at * HD + d;
                    const uint4* w = reinterpret_cast<const uint4*>(src);      // (rows of a pool lie on 16 bytes)
                    alignas(16) KVT k8[8];
#pragma unroll
                    for (int e = 0; e < (int)sizeof(KVT) / 2; ++e) reinterpret_cast<uint4*>(k8)[e] = w[e];
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = Elem<KVT>::get(k8, e);
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) s = fmaf(Elem<RT>::get(qp, d + e), x[e], s);
            }
            s *= scale;
        }
        float mn = s;
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, x));
        mn = fmaxf(top, mn);
        const float ref = mn == -INFINITY ? 0.f : mn, f = top == mn ? 1.f : expf(top - ref), w = sees ? expf(s - ref) : 0.f;
        top = mn;
        sum = sum * f + warp_sum(w);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] *= f;
        // eight rows of V on their way at once; those that the row does not see (or of page 0, where there is no second page) become zeros
        for (int j0 = 0; j0 < 32; j0 += 8) {
            constexpr int W = Q4 ? 1 : E * (int)sizeof(KVT) / 4;
            uint32_t x[8][W];
            float one[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const size_t at = ((size_t)__shfl_sync(0xffffffffu, id, j0 + u) * p.c.kv_heads + kvh) * kKvBlock + (j0 + u) % kKvBlock;
                if constexpr (Q4) {
                    const unsigned char* codes = static_cast<const unsigned char*>(p.c.vpool) + at * (HD / 2) + lane * E / 2;
                    x[u][0] = E == 4 ? *reinterpret_cast<const unsigned short*>(codes) : *codes;
                    one[u] = e4m3_to_f32(p.c.vscale[at * (HD / 16) + lane * E / 16]);
                } else {
                    const uint32_t* src = reinterpret_cast<const uint32_t*>(static_cast<const KVT*>(p.c.vpool) + at * HD + lane * E);
#pragma unroll
                    for (int e = 0; e < W; ++e) x[u][e] = src[e];
                }
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float wj = __shfl_sync(0xffffffffu, w, j0 + u);
                const bool use = seen >> (j0 + u) & 1u;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    float y;
                    if constexpr (Q4) y = e2m1_value(x[u][0] >> (4 * e)) * one[u];
                    else if constexpr (sizeof(KVT) == 2) y = __uint_as_float(e % 2 ? x[u][e / 2] & 0xffff0000u : x[u][e / 2] << 16);
                    else y = __uint_as_float(x[u][e]);
                    o[e] = use ? fmaf(wj, y, o[e]) : o[e];
                }
            }
        }
        bool none = sum != sum;                  // a NaN stays one
        if (!none) {
            none = true;
#pragma unroll
            for (int e = 0; e < E; ++e) none = none && o[e] != o[e];
        }
        if (__all_sync(0xffffffffu, none)) break;
    }
    RT* op = static_cast<RT*>(p.out) + (size_t)row * p.out_stride + (size_t)h * HD + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        float y = any ? o[e] / sum * p.c.v_scale : 0.f;
        if (p.gate && any) y *= p.gate[(size_t)row * p.heads * HD + (size_t)h * HD + lane * E + e];
        Elem<RT>::put(op, e, y);
    }
}

// A launch that need not wait for the kernel before it: that one says when (pdl_launch_dependents), and this one waits itself for its end (pdl_wait)
template <typename... KArgs>
static cudaError_t launch_after(void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, cudaStream_t st, KArgs... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace mlb
