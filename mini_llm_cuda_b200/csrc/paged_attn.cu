// Attention of new rows over a caller's paged K/V cache (mlb_op_attn_paged): fp32, bf16 or 4-bit pages, a causal mask with an optional
// window and first positions that stay visible, one to many rows per sequence.
#include <algorithm>
#include <type_traits>

#include "paged.cuh"

namespace mlb {

namespace {

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// ---- one row, one head, by one warp, straight from the formula --------------------------------------------------------
// A product with a probability that is not of the row's own positions does not happen here, so infinities and NaN outside of them cannot
// reach the row, and an infinite score or value gives what the formula gives. The matrix-core kernels redo a row here whose result is
// not finite: there a probability of 0 times an infinity, or a piece of an infinite number, is a NaN.
template <typename KVT, typename RT, int HD>
__device__ __noinline__ void careful_row(const AttnPagedParams& p, int b, int pos, int row, int h) {
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

template <typename KVT, typename RT, int HD>
__global__ void __launch_bounds__(256) attn_paged_rows_kernel(const __grid_constant__ AttnPagedParams p) {
    const int warp = (blockIdx.x * 256 + threadIdx.x) >> 5, row = warp / p.heads, h = warp % p.heads;
    if (row >= p.r.rows) return;
    int b = row;
    if (p.r.row_start) {
        b = 0;
        while (b + 1 < p.r.batch && p.r.row_start[b + 1] <= row) ++b;
    } else if (b >= p.r.batch) {
        return;
    }
    const PagedSeq s = paged_seq(p.r, p.c.pt_stride, b, true);
    if (row < s.r0 || row >= s.r0 + s.n) return;
    careful_row<KVT, RT, HD>(p, b, s.len - s.n + row - s.r0, row, h);
}

template <typename KVT, typename RT>
cudaError_t rows_launch(const AttnPagedParams& p, int hd, cudaStream_t st) {
    const unsigned ctas = (unsigned)(((long long)p.r.rows * p.heads + 7) / 8);
    if (hd == 64) attn_paged_rows_kernel<KVT, RT, 64><<<ctas, 256, 0, st>>>(p);
    else attn_paged_rows_kernel<KVT, RT, 128><<<ctas, 256, 0, st>>>(p);
    return cudaGetLastError();
}

}  // namespace

size_t attn_paged_part_bytes(int sm_count) { return (size_t)sm_count * 16 * 2 * 8 * 130 * 4; }

cudaError_t attn_paged_launch(const AttnPagedParams& p, int dtype, int row_dtype, int head_dim, int sm_count, cudaStream_t st) {
    const bool f = row_dtype == MLB_DT_F32;
    if (dtype == MLB_DT_F32) return f ? rows_launch<float, float>(p, head_dim, st) : rows_launch<float, bf16_t>(p, head_dim, st);
    if (dtype == MLB_DT_BF16) return f ? rows_launch<bf16_t, float>(p, head_dim, st) : rows_launch<bf16_t, bf16_t>(p, head_dim, st);
    return f ? rows_launch<fp4_t, float>(p, head_dim, st) : rows_launch<fp4_t, bf16_t>(p, head_dim, st);
}

}  // namespace mlb
