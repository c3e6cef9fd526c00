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
// not finite: there a probability of 0 times an infinity, or a piece of an infinite number, is a NaN.
template <typename KVT, typename RT, int HD>
static __device__ __noinline__ void careful_row(const AttnPagedParams& p, int b, int pos, int row, int h) {
    constexpr int E = HD / 32;                   // dims of a lane
    const int lane = threadIdx.x & 31, kvh = h / p.group;
    float q[E], o[E], top = -INFINITY, sum = 0.f;
    const RT* qp = static_cast<const RT*>(p.q) + (size_t)row * p.q_stride + (size_t)h * HD + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        q[e] = Elem<RT>::get(qp, e);
        o[e] = 0.f;
    }
    auto get = [&](bool k, size_t at, float (&x)[E]) {      // this lane's dims of pool row `at`
        if constexpr (sizeof(KVT) == 1) {
            const unsigned char* codes = static_cast<const unsigned char*>(k ? p.c.kpool : p.c.vpool) + at * (HD / 2) + lane * E / 2;
            const float s = e4m3_to_f32((k ? p.c.kscale : p.c.vscale)[at * (HD / 16) + lane * E / 16]);
#pragma unroll
            for (int e = 0; e < E; e += 2) {
                x[e] = e2m1_value(codes[e / 2] & 15) * s;
                x[e + 1] = e2m1_value(codes[e / 2] >> 4) * s;
            }
        } else {
            const KVT* src = static_cast<const KVT*>(k ? p.c.kpool : p.c.vpool) + at * HD + lane * E;
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = Elem<KVT>::get(src, e);
        }
    };
    const PagedSpan span = paged_span(p, pos, pos);
    const float scale = p.scale * p.c.k_scale;
    bool any = false;
    for (int v = 0; v < span.count; ++v) {
        const int pg = span.page(v), id = paged_page(p.c, p.r.err, b, pg, 0);
        const size_t base = ((size_t)id * p.c.kv_heads + kvh) * kKvBlock;
        for (int j = 0; j < kKvBlock; ++j) {
            if (!paged_sees(p, pos, pg * kKvBlock + j)) continue;
            float x[E], s = 0.f;
            get(true, base + j, x);
#pragma unroll
            for (int e = 0; e < E; ++e) s = fmaf(q[e], x[e], s);
            s = warp_sum(s) * scale;
            any = true;
            const float mn = fmaxf(top, s), ref = mn == -INFINITY ? 0.f : mn;
            const float f = top == mn ? 1.f : expf(top - ref), w = expf(s - ref);
            top = mn;
            sum = sum * f + w;
            get(false, base + j, x);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = fmaf(w, x[e], o[e] * f);
        }
    }
    RT* op = static_cast<RT*>(p.out) + (size_t)row * p.out_stride + (size_t)h * HD + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        float y = any ? o[e] / sum * p.c.v_scale : 0.f;
        if (p.gate) y *= p.gate[(size_t)row * p.heads * HD + (size_t)h * HD + lane * E + e];
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
