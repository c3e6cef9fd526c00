// Attention of new rows over a caller's paged K/V cache (mlb_op_attn_paged): fp32, bf16 or 4-bit pages, a causal mask with an optional
// window and first positions that stay visible, one to many rows per sequence.
#include <algorithm>
#include <type_traits>

#include "paged_prompt.h"
#include "paged_row.cuh"
#include "ring.cuh"

namespace mlb {

namespace {

// ---- blocks of up to eight rows on matrix cores -------------------------------------------------------------------------
// A warp takes pages of 16 positions of one K/V head for a block of up to 8 rows (new tokens x the query heads of the K/V head):
//   S[16 positions][8 rows] = K Q^T      A = K, B = Q^T,  m16n8k16
//   O^T[dims][8 rows] += V^T P^T         A = V^T, B = P^T
// fp32 and bf16 pages go straight to registers: dims of a dot product and positions of a sum may come in any order, so a lane loads 16
// bytes of a K row and uses them as its elements of two (fp32: one, 4 bits: eight) k-steps, and 16 bytes each of four V rows whose
// 16-bit halves it pairs up with byte permutes. S lies with positions along the lanes and rows within them, as O does: a running maximum
// and its rescaling need no exchange between lanes but the maximum itself, and that only when a score passes the old one by 2^8; P is
// turned round by movmatrix.
// fp32 numbers are taken in pieces whose products are exact: fp32 queries, K, V and probabilities in three bf16, probabilities of bf16 rows in two. Products of
// pieces below 2^-24 of the whole are left out. Matrix cores cut off where they add, at the size of what they add to: the products of pieces behind the first have
// sums of their own in a score, and with fp32 rows a page's values are summed by themselves and added to the pages' before it in fp32 (error against 64 bits 2e-7 to
// 5e-7 of the answer, 5e-7 to 2e-6 with everything in one sum, at 0 to 8 % of the time). 4-bit codes times their e4m3 scale are exact halves, to which the conversion instruction brings them, and meet
// queries as halves (fp32: two of them, bf16: one), the row scaled by a power of two to lie within their range.
// A probability may have any magnitude: where one position outweighs the rest and brings next to nothing (the first one does both in trained models) the answer
// is what the rest add up to. bf16 has that range. Halves, which the codes of V come to at less cost, have 11 bits from 2^-14 to 2^15: so over 4-bit
// pages the codes of V are widened to bf16 too, but for up to four bf16 rows, whose probabilities are halves in two bands (page_values).
constexpr int kSplitWarps = 8;
constexpr float kLazy = 8.f;         // log2 of how far a score may pass the running maximum before it is moved

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <int BYTES>
__device__ __forceinline__ void cp_async(uint32_t to, const void* from) {
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
    uint32_t y;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
    return y;
}
// N bf16 (or half) pairs whose sum is the pair (x, y) to 8 N bits (11 N, of halves no finer than 2^-25)
template <bool HALF = false, int N>
__device__ __forceinline__ void pieces(float x, float y, uint32_t (&o)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        o[i] = HALF ? f32x2_to_f16(x, y) : f32x2_to_bf16(x, y);
        if (i + 1 < N) {
            x -= HALF ? f16_lo(o[i]) : __uint_as_float(o[i] << 16);
            y -= HALF ? f16_hi(o[i]) : __uint_as_float(o[i] & 0xffff0000u);
        }
    }
}

// What a lane (g = lane / 4, j = lane % 4) holds of a page's K and V rows. A k-step's slots 0, 1 are k = 2j, 2j + 1, slots 2, 3 k = 2j + 8, 2j + 9;
// dim() says which dim stands there. V: block vb of the lane's dims and M-tile mt within it hold dims vdim() and the next one.
template <typename KVT, int HD> struct PageFrag;

template <int HD>
struct PageFrag<bf16_t, HD> {
    static constexpr int KP = 1;                             // pieces of K and V
    static constexpr bool Q4 = false;
    uint4 k[2][HD / 32], v[HD / 64][4];
    __device__ static int dim(int ks, int j, int slot) { return ks / 2 * 32 + j * 8 + ks % 2 * 4 + slot; }
    __device__ static int vdim(int mt, int g) { return mt / 4 * 64 + g * 8 + mt % 4 * 2; }
    __device__ __forceinline__ void load_k(const PagedCache& c, size_t base, int g, int j) {
        const uint4* p = reinterpret_cast<const uint4*>(static_cast<const bf16_t*>(c.kpool) + base * HD);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int b = 0; b < HD / 32; ++b) k[t][b] = __ldg(p + (t * 8 + g) * (HD / 8) + b * 4 + j);
    }
    __device__ __forceinline__ void load_v(const PagedCache& c, size_t base, int g, int j) {
        const uint4* p = reinterpret_cast<const uint4*>(static_cast<const bf16_t*>(c.vpool) + base * HD);
#pragma unroll
        for (int b = 0; b < HD / 64; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[b][i] = __ldg(p + (2 * j + (i & 1) + (i & 2) * 4) * (HD / 8) + b * 8 + g);
    }
    __device__ __forceinline__ void hide_v(int i) {          // row i of the lane's four holds no number that may be used
#pragma unroll
        for (int b = 0; b < HD / 64; ++b) v[b][i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void k_operand(int ks, uint32_t (&a)[1][4]) const {
        const uint4 x = k[0][ks / 2], y = k[1][ks / 2];
        a[0][0] = ks % 2 ? x.z : x.x; a[0][1] = ks % 2 ? y.z : y.x; a[0][2] = ks % 2 ? x.w : x.y; a[0][3] = ks % 2 ? y.w : y.y;
    }
    __device__ __forceinline__ void v_operand(int mt, uint32_t (&a)[1][4]) const {
        auto word = [&](int i) {
            const uint4& x = v[mt / 4][i];
            return mt % 4 == 0 ? x.x : mt % 4 == 1 ? x.y : mt % 4 == 2 ? x.z : x.w;
        };
        a[0][0] = __byte_perm(word(0), word(1), 0x5410); a[0][1] = __byte_perm(word(0), word(1), 0x7632);
        a[0][2] = __byte_perm(word(2), word(3), 0x5410); a[0][3] = __byte_perm(word(2), word(3), 0x7632);
    }
};

template <int HD>
struct PageFrag<float, HD> {
    static constexpr int KP = 3;
    static constexpr bool Q4 = false;
    float4 k[2][HD / 16], v[HD / 32][4];
    __device__ static int dim(int ks, int j, int slot) { return ks * 16 + j * 4 + slot; }
    __device__ static int vdim(int mt, int g) { return mt / 2 * 32 + g * 4 + mt % 2 * 2; }
    __device__ __forceinline__ void load_k(const PagedCache& c, size_t base, int g, int j) {
        const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(c.kpool) + base * HD);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int b = 0; b < HD / 16; ++b) k[t][b] = __ldg(p + (t * 8 + g) * (HD / 4) + b * 4 + j);
    }
    __device__ __forceinline__ void load_v(const PagedCache& c, size_t base, int g, int j) {
        const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(c.vpool) + base * HD);
#pragma unroll
        for (int b = 0; b < HD / 32; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[b][i] = __ldg(p + (2 * j + (i & 1) + (i & 2) * 4) * (HD / 4) + b * 8 + g);
    }
    __device__ __forceinline__ void hide_v(int i) {
#pragma unroll
        for (int b = 0; b < HD / 32; ++b) v[b][i] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    __device__ __forceinline__ void k_operand(int ks, uint32_t (&a)[3][4]) const {
        uint32_t w[4][3];
        pieces(k[0][ks].x, k[0][ks].y, w[0]);
        pieces(k[1][ks].x, k[1][ks].y, w[1]);
        pieces(k[0][ks].z, k[0][ks].w, w[2]);
        pieces(k[1][ks].z, k[1][ks].w, w[3]);
#pragma unroll
        for (int i = 0; i < 3; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) a[i][e] = w[e][i];
    }
    __device__ __forceinline__ void v_operand(int mt, uint32_t (&a)[3][4]) const {
        uint32_t w[4][3];
#pragma unroll
        for (int h = 0; h < 4; ++h) {                        // a0, a1: keys 2j, 2j + 1 of the two dims; a2, a3: keys 2j + 8, 2j + 9
            const float4 &x = v[mt / 2][h / 2 * 2], &y = v[mt / 2][h / 2 * 2 + 1];
            const float u = mt % 2 ? (h % 2 ? x.w : x.z) : (h % 2 ? x.y : x.x), z = mt % 2 ? (h % 2 ? y.w : y.z) : (h % 2 ? y.y : y.x);
            pieces(u, z, w[h]);
        }
#pragma unroll
        for (int i = 0; i < 3; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) a[i][e] = w[e][i];
    }
};

template <int HD>
struct PageFrag<fp4_t, HD> {
    static constexpr int KP = 1;
    static constexpr bool Q4 = true;
    static constexpr int KW = HD / 32, VW = HD / 64;         // words of codes of a K row per lane, of a V row
    uint32_t k[2][KW], ks_[2], v[4][VW], vs[2];
    __device__ static int dim(int ks, int j, int slot) { return j * (HD / 4) + ks * 4 + slot; }
    __device__ static int vdim(int mt, int g) { return g * (HD / 8) + mt * 2; }
    // A page in shared memory: codes of K, of V (of 128 dims, with the 16-byte pieces of a row moved by row / 2, against bank conflicts), scales of K, of V
    static constexpr int kCodes = 16 * HD / 2, kScales = HD, kBytes = 2 * (kCodes + kScales);
    __device__ static void copy(const PagedCache& c, size_t base, uint32_t to, int lane) {
        const unsigned char *k = static_cast<const unsigned char*>(c.kpool) + base * (HD / 2) + lane * 16, *v = static_cast<const unsigned char*>(c.vpool) + base * (HD / 2) + lane * 16;
#pragma unroll
        for (int i = 0; i < HD / 64; ++i) {
            const int piece = lane + 32 * i, row = piece / (HD / 32), ch = piece % (HD / 32);
            cp_async<16>(to + piece * 16, k + i * 512);
            cp_async<16>(to + kCodes + row * (HD / 2) + (HD == 128 ? ch ^ (row >> 1 & 3) : ch) * 16, v + i * 512);
        }
        if (lane < kScales / 4) {
            cp_async<4>(to + 2 * kCodes + lane * 4, c.kscale + base * (HD / 16) + lane * 4);
            cp_async<4>(to + 2 * kCodes + kScales + lane * 4, c.vscale + base * (HD / 16) + lane * 4);
        }
    }
    __device__ __forceinline__ void read_k(const unsigned char* page, int g, int j) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int row = t * 8 + g;
            if constexpr (HD == 128) {
                const uint4 x = *reinterpret_cast<const uint4*>(page + row * 64 + j * 16);
                k[t][0] = x.x; k[t][1] = x.y; k[t][2 % KW] = x.z; k[t][3 % KW] = x.w;
                ks_[t] = *reinterpret_cast<const unsigned short*>(page + 2 * kCodes + row * 8 + j * 2);
            } else {
                const uint2 x = *reinterpret_cast<const uint2*>(page + row * 32 + j * 8);
                k[t][0] = x.x; k[t][1] = x.y;
                ks_[t] = page[2 * kCodes + row * 4 + j];
            }
        }
    }
    __device__ __forceinline__ void read_v(const unsigned char* page, int g, int j) {
        uint32_t b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = 2 * j + (i & 1) + (i & 2) * 4;
            if constexpr (HD == 128) {
                const uint2 x = *reinterpret_cast<const uint2*>(page + kCodes + row * 64 + ((g >> 1) ^ j) * 16 + (g & 1) * 8);
                v[i][0] = x.x; v[i][1 % VW] = x.y;
                b[i] = page[2 * kCodes + kScales + row * 8 + g];
            } else {
                v[i][0] = *reinterpret_cast<const uint32_t*>(page + kCodes + row * 32 + g * 4);
                b[i] = page[2 * kCodes + kScales + row * 4 + g / 2];
            }
        }
        vs[0] = b[0] | b[1] << 8;
        vs[1] = b[2] | b[3] << 8;
    }
    __device__ __forceinline__ void hide_v(int i) {          // (codes are numbers, but a scale's byte may be a NaN)
#pragma unroll
        for (int w = 0; w < VW; ++w) v[i][w] = 0;
        vs[i / 2] &= i % 2 ? 0x00ffu : 0xff00u;
    }
    // all k-steps at once: h[t][i] = two dims of row t * 8 + g
    __device__ __forceinline__ void widen_k(uint32_t (&h)[2][HD / 8]) const {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const uint32_t s = e4m3x2_to_f16(ks_[t]), s0 = __byte_perm(s, s, 0x1010), s1 = __byte_perm(s, s, 0x3232);
#pragma unroll
            for (int w = 0; w < KW; ++w) {
                uint32_t o[4];
                e2m1x8_to_f16(k[t][w], o);
#pragma unroll
                for (int i = 0; i < 4; ++i) h[t][w * 4 + i] = hmul2(o[i], w < 2 ? s0 : s1);
            }
        }
    }
};

// Scores of a page: s[0..1] position g of rows 2j, 2j + 1, s[2..3] position g + 8. `qf` holds the rows' pieces as B operands: [piece][k-step][lane].
template <typename KVT, int HD, int QP>
__device__ __forceinline__ void page_scores(const PageFrag<KVT, HD>& f, const uint2* qf, int lane, float (&s)[4]) {
    using F = PageFrag<KVT, HD>;
    float t[4] = {0.f, 0.f, 0.f, 0.f}, low[4] = {0.f, 0.f, 0.f, 0.f};       // two chains of products, and those of pieces behind the first
    s[0] = s[1] = s[2] = s[3] = 0.f;
    if constexpr (F::Q4) {
        uint32_t h[2][HD / 8];
        f.widen_k(h);
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
            for (int i = 0; i < QP; ++i) {
                const uint2 b = qf[(i * (HD / 16) + ks) * 32 + lane];
                mma_f16(i > 0 ? low : ks % 2 ? t : s, h[0][2 * ks], h[1][2 * ks], h[0][2 * ks + 1], h[1][2 * ks + 1], b.x, b.y);
            }
    } else {
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) {
            uint32_t a[F::KP][4];
            f.k_operand(ks, a);
#pragma unroll
            for (int i = 0; i < QP; ++i) {
                const uint2 b = qf[(i * (HD / 16) + ks) * 32 + lane];
#pragma unroll
                for (int k = 0; k < F::KP; ++k)
                    if (i + k < 3) mma_bf16(i + k > 0 ? low : ks % 2 ? t : s, a[k][0], a[k][1], a[k][2], a[k][3], b.x, b.y);
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] = QP > 1 || F::KP > 1 ? s[e] + t[e] + low[e] : s[e] + t[e];
}

// Up to four bf16 rows over 4-bit pages leave half of an MMA's columns empty. The first four hold a row's weights times 2^13 from 2^-13 on, the others the row
// again (PAIR, lanes with j >= 2) with those below, times 2^37: 52 bits of range as halves for one MMA. Relative to the largest weight, which
// stands at 2^13 to 2^15 there, all down to 2^-51 have 11 bits, and those below 2^-62 are lost. 128 sequences of up to 8000 positions, 4 rows each: 144 us;
// with V in bf16 and two pieces 174, one piece 159 (8 bits); 139 with halves alone, which lost what lay below 2^-25. Of 8 rows each, which have bf16: 177.
constexpr float kPairUp = 8192.f, kPairLow = 137438953472.f, kPairLazy = 2.f;      // 2^13, 2^37; log2 of how far a score may pass the running maximum

// acc[mt]: dims vdim(mt, g) of rows 2j, 2j + 1 in [0], [1], the next dim in [2], [3] (4-bit pages in bf16: a 256th of them, as widen_codes has it)
template <typename KVT, int HD, int PIECES, bool PAIR>
__device__ __forceinline__ void page_values(const PageFrag<KVT, HD>& f, const float (&w)[4], float (&acc)[HD / 16][4]) {
    using F = PageFrag<KVT, HD>;
    constexpr int PP = PAIR ? 1 : PIECES;
    uint32_t p0[PP], p1[PP];
    if constexpr (PAIR) {
        // (a weight next to 2^-13 is the same number in both lanes and rounds to the same 11 bits in both bands, and so falls to one)
        const bool second = threadIdx.x & 2;
        const uint32_t flip = second ? 0xffffffffu : 0u, at = second ? 0x68006800u : 0x08000800u;      // 2^11, 2^-13
        const float up = second ? kPairLow : kPairUp;
        auto band = [&](float x, float y) {
            const uint32_t h = f32x2_to_f16(x * up, y * up);
            return h & (__hge2_mask(*reinterpret_cast<const __half2*>(&h), *reinterpret_cast<const __half2*>(&at)) ^ flip);
        };
        p0[0] = band(w[0], w[1]);
        p1[0] = band(w[2], w[3]);
    } else {
        pieces(w[0], w[1], p0);
        pieces(w[2], w[3], p1);
    }
#pragma unroll
    for (int i = 0; i < PP; ++i) {
        p0[i] = movmatrix(p0[i]);
        p1[i] = movmatrix(p1[i]);
    }
    if constexpr (PAIR) {
        const uint32_t s0 = e4m3x2_to_f16(f.vs[0]), s1 = e4m3x2_to_f16(f.vs[1]);
#pragma unroll
        for (int w8 = 0; w8 < F::VW; ++w8) {
            // codes of one dim and two neighbouring rows side by side, of even dims, of odd ones
            uint32_t h[4][4];
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                const uint32_t x = f.v[i][w8], y = f.v[i + 1][w8];
                e2m1x8_to_f16((x & 0x0f0f0f0fu) | (y << 4 & 0xf0f0f0f0u), h[i]);
                e2m1x8_to_f16((x >> 4 & 0x0f0f0f0fu) | (y & 0xf0f0f0f0u), h[i + 1]);
            }
#pragma unroll
            for (int m = 0; m < 4; ++m)
                mma_f16(acc[w8 * 4 + m], hmul2(h[0][m], s0), hmul2(h[1][m], s0), hmul2(h[2][m], s1), hmul2(h[3][m], s1), p0[0], p1[0]);
        }
    } else if constexpr (F::Q4) {
        const uint32_t h0 = e4m3x2_to_f16(f.vs[0]), h1 = e4m3x2_to_f16(f.vs[1]);
        const uint32_t s0 = f32x2_to_bf16(f16_lo(h0) * kScaleUp, f16_hi(h0) * kScaleUp), s1 = f32x2_to_bf16(f16_lo(h1) * kScaleUp, f16_hi(h1) * kScaleUp);
#pragma unroll
        for (int w = 0; w < 2 * F::VW; ++w) {
            // four dims of two neighbouring rows, the one's codes under the other's: widen_codes puts a dim's two together
            const int sel = w % 2 ? 0x7632 : 0x5410;
            const uint4 x = widen_codes(__byte_perm(f.v[0][w / 2], f.v[1][w / 2], sel), s0), y = widen_codes(__byte_perm(f.v[2][w / 2], f.v[3][w / 2], sel), s1);
            float own[2][4] = {};                            // the page's, smallest products first
#pragma unroll
            for (int i = PP - 1; i >= 0; --i) {
                mma_bf16(PP == 3 ? own[0] : acc[w * 2], x.x, x.y, y.x, y.y, p0[i], p1[i]);
                mma_bf16(PP == 3 ? own[1] : acc[w * 2 + 1], x.z, x.w, y.z, y.w, p0[i], p1[i]);
            }
            if constexpr (PP == 3)
#pragma unroll
                for (int e = 0; e < 4; ++e) { acc[w * 2][e] += own[0][e]; acc[w * 2 + 1][e] += own[1][e]; }
        }
    } else {
#pragma unroll
        for (int mt = 0; mt < HD / 16; ++mt) {
            uint32_t a[F::KP][4];
            float own[4] = {};
            f.v_operand(mt, a);
#pragma unroll
            for (int o = 2; o >= 0; --o)                     // pieces o - k of the weights and k of V
#pragma unroll
                for (int k = 0; k < F::KP; ++k)
                    if (k <= o && o - k < PP) mma_bf16(PP == 3 ? own : acc[mt], a[k][0], a[k][1], a[k][2], a[k][3], p0[o - k], p1[o - k]);
            if constexpr (PP == 3)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[mt][e] += own[e];
        }
    }
}

// A block of rows of one K/V head: rows first .. first + count - 1 of the sequence's (token, head) pairs, token by token
struct Block {
    int b, kvh, first, count;
    PagedSeq s;
};

template <typename RT, int QP, int HD, typename F>
__device__ __forceinline__ void pack_queries(const AttnPagedParams& p, const Block& k, bool pair, uint2* qf, float* qscale, int lane) {
    const int g = lane >> 2, j = lane & 3;                   // the B operand's column is a row of the block
    const int i = pair ? g & 3 : g;
    const bool in = i < k.count;
    const int r = k.first + (in ? i : 0), row = k.s.r0 + r / p.group, h = k.kvh * p.group + r % p.group;
    const RT* q = static_cast<const RT*>(p.q) + (size_t)row * p.q_stride + (size_t)h * HD;
    // four neighbouring dims for each k-step, all on their way at once
    float x[HD / 16][4];
    const bool vec = reinterpret_cast<uintptr_t>(q) % (4 * sizeof(RT)) == 0;
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) {
        const RT* src = q + F::dim(ks, j, 0);
        if (!in) {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[ks][e] = 0.f;
        } else if (!vec) {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[ks][e] = Elem<RT>::get(src, e);
        } else if constexpr (sizeof(RT) == 4) {
            const float4 w = __ldg(reinterpret_cast<const float4*>(src));
            x[ks][0] = w.x; x[ks][1] = w.y; x[ks][2] = w.z; x[ks][3] = w.w;
        } else {
            const uint2 w = __ldg(reinterpret_cast<const uint2*>(src));
            x[ks][0] = __uint_as_float(w.x << 16); x[ks][1] = __uint_as_float(w.x & 0xffff0000u);
            x[ks][2] = __uint_as_float(w.y << 16); x[ks][3] = __uint_as_float(w.y & 0xffff0000u);
        }
    }
    float up = 1.f, down = 1.f;
    if (F::Q4) {
        // a power of two that brings the row's largest magnitude to 256 .. 512, if it is a number
        float top = 0.f;
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
            for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(x[ks][e]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = max(-100, min(100, 8 - ((int)(__float_as_uint(top) >> 23) - 127)));
        up = __uint_as_float((uint32_t)(127 + e) << 23);
        down = __uint_as_float((uint32_t)(127 - e) << 23);
    }
    if (j == 0) qscale[g] = p.scale * p.c.k_scale * 1.4426950408889634f * down;
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) {
        uint32_t lo[QP], hi[QP];
        pieces<F::Q4>(x[ks][0] * up, x[ks][1] * up, lo);
        pieces<F::Q4>(x[ks][2] * up, x[ks][3] * up, hi);
#pragma unroll
        for (int i = 0; i < QP; ++i) qf[(i * (HD / 16) + ks) * 32 + lane] = make_uint2(lo[i], hi[i]);
    }
}

template <typename KVT, typename RT, int HD>
struct SplitShape {
    using F = PageFrag<KVT, HD>;
    static constexpr int QP = sizeof(RT) == 2 ? 1 : F::Q4 ? 2 : 3;
    static constexpr int PP = sizeof(RT) == 4 ? 3 : 2;
    static constexpr bool MAY_PAIR = F::Q4 && PP == 2;
    __device__ static bool pair(int count) { return MAY_PAIR && count <= 4; }
    static constexpr int QWORDS = QP * (HD / 16) * 32;       // uint2 of a warp's queries
    static constexpr int W = HD + 2;                         // floats of a row's partial result: its sums, maximum, total
    static constexpr int PART = 8 * W;
};
__host__ __device__ constexpr int split_part_floats(int hd) { return 8 * (hd + 2); }

// How a warp gets the pages v, v + step, .. < v1: into registers, K of the next one while this one's V is weighed. Made before the queries are
// packed, so that the first loads are under way.
template <typename KVT, int HD>
struct PageSource {
    static constexpr int kRing = 0;              // bytes of shared memory
    const AttnPagedParams& p;
    const Block& k;
    const PagedSpan& span;
    const int v1, step;
    PageFrag<KVT, HD> f;
    int id = 0, next = 0;
    __device__ __forceinline__ size_t base(int x) const { return ((size_t)x * p.c.kv_heads + k.kvh) * kKvBlock; }
    __device__ __forceinline__ PageSource(const AttnPagedParams& p_, const Block& k_, const PagedSpan& span_, int v, int v1_, int step_, unsigned char*)
        : p(p_), k(k_), span(span_), v1(v1_), step(step_) {
        if (v >= v1) return;
        id = paged_page(p.c, p.r.err, k.b, span.page(v), 0);
        if (v + step < v1) next = paged_page(p.c, p.r.err, k.b, span.page(v + step), 0);
        f.load_k(p.c, base(id), (threadIdx.x & 31) >> 2, threadIdx.x & 3);
    }
    __device__ __forceinline__ void begin(int, int g, int j) { f.load_v(p.c, base(id), g, j); }      // page v
    __device__ __forceinline__ void k_used(int v, int g, int j) {
        if (v + step < v1) f.load_k(p.c, base(next), g, j);
        id = next;
        if (v + 2 * step < v1) next = paged_page(p.c, p.r.err, k.b, span.page(v + 2 * step), 0);
    }
    __device__ __forceinline__ void want_v(int, int) {}
    __device__ __forceinline__ void end() {}
};
// 4-bit pages are small (2.3 KB for 16 positions of K and V, 128 dims): a warp has up to kStages - 1 on their way to a ring in shared memory, and one load
// brings the ids of 32. (In registers, one page and a half: 2.6 of 7 cycles between a warp's instructions went by waiting for them.)
template <int HD>
struct PageSource<fp4_t, HD> {
    using F = PageFrag<fp4_t, HD>;
    static constexpr int kStages = 4, kRing = kStages * F::kBytes;
    const AttnPagedParams& p;
    const Block& k;
    const PagedSpan& span;
    const int v1, step;
    unsigned char* const ring;
    F f;
    int ahead, count = 0, used = 0;              // next page to bring; pages brought, and used
    int ids = 0, more_ids = 0;                   // of 32 pages, a lane each, and of the 32 after these
    __device__ __forceinline__ int load_ids(int v) const {
        v += (int)(threadIdx.x & 31) * step;
        return v < v1 ? paged_page(p.c, p.r.err, k.b, span.page(v), 0) : 0;
    }
    __device__ __forceinline__ void bring() {
        if (ahead < v1) {
            const int id = __shfl_sync(0xffffffffu, ids, count & 31);
            F::copy(p.c, ((size_t)id * p.c.kv_heads + k.kvh) * kKvBlock, smem_u32(ring) + (uint32_t)(count % kStages) * F::kBytes, threadIdx.x & 31);
            ahead += step;
            if ((++count & 31) == 0) {
                ids = more_ids;
                more_ids = load_ids(ahead + 32 * step);
            }
        }
        cp_async_commit();                       // (an empty group too, so that waits count pages)
    }
    __device__ __forceinline__ PageSource(const AttnPagedParams& p_, const Block& k_, const PagedSpan& span_, int v, int v1_, int step_, unsigned char* ring_)
        : p(p_), k(k_), span(span_), v1(v1_), step(step_), ring(ring_), ahead(v) {
        ids = load_ids(v);
        more_ids = load_ids(v + 32 * step);
#pragma unroll
        for (int i = 0; i < kStages - 1; ++i) bring();
    }
    __device__ __forceinline__ const unsigned char* page() const { return ring + used % kStages * F::kBytes; }
    __device__ __forceinline__ void begin(int, int g, int j) {
        cp_async_wait<kStages - 2>();
        __syncwarp();                            // all lanes' pieces are there, and the page before has been used by all
        bring();
        f.read_k(page(), g, j);
    }
    __device__ __forceinline__ void k_used(int, int, int) {}
    __device__ __forceinline__ void want_v(int g, int j) {
        f.read_v(page(), g, j);
        ++used;
    }
    __device__ __forceinline__ void end() {
        cp_async_wait<0>();
        __syncwarp();
    }
};
// The pages v, v + step, .. < v1 of a span for a block; results in acc, m (log2 of the reference of the weights) and l
template <typename KVT, typename RT, int HD, bool PAIR>
__device__ __forceinline__ void walk_rows(const AttnPagedParams& p, const Block& k, const PagedSpan& span, int v, int v1, int step, PageSource<KVT, HD>& src,
                                          const uint2* qf, const float* qscale, float (&acc)[HD / 16][4], float (&m)[2], float (&l)[2]) {
    using S = SplitShape<KVT, RT, HD>;
    const int lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3;
#pragma unroll
    for (int t = 0; t < HD / 16; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][e] = 0.f;
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
    if (v >= v1) {
        src.end();
        return;
    }
    const int pos0 = k.s.len - k.s.n;
    int pos[2];
    const int i0 = PAIR ? 2 * j & 3 : 2 * j;                 // this lane's first row
    pos[0] = i0 < k.count ? pos0 + (k.first + i0) / p.group : -1;
    pos[1] = i0 + 1 < k.count ? pos0 + (k.first + i0 + 1) / p.group : -1;
    const int low = pos0 + k.first / p.group, high = pos0 + (k.first + k.count - 1) / p.group;      // positions of the block's rows
    const float c0 = qscale[2 * j], c1 = qscale[2 * j + 1];
    PageFrag<KVT, HD>& f = src.f;
#pragma unroll 1
    for (; v < v1; v += step) {
        const int key0 = span.page(v) * kKvBlock;
        src.begin(v, g, j);
        float s[4];
        page_scores<KVT, HD, S::QP>(f, qf, lane, s);
        src.k_used(v, g, j);
        s[0] *= c0; s[1] *= c1; s[2] *= c0; s[3] *= c1;
        src.want_v(g, j);
        if (key0 + kKvBlock - 1 > low || (p.window > 0 && key0 <= high - p.window && key0 + kKvBlock > p.sinks)) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (!paged_sees(p, pos[e & 1], key0 + g + (e & 2) * 4)) s[e] = -INFINITY;
            // 0 times what is no number is no number: values that no row sees become zeros
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = key0 + 2 * j + (i & 1) + (i & 2) * 4;
                if (key > high || (p.window > 0 && key <= low - p.window && key >= p.sinks)) f.hide_v(i);
            }
        }
        const float t0 = fmaxf(s[0], s[2]), t1 = fmaxf(s[1], s[3]);
        constexpr float lazy = PAIR ? kPairLazy : kLazy;
        if (__any_sync(0xffffffffu, t0 > m[0] + lazy || t1 > m[1] + lazy)) {
            float n0 = fmaxf(m[0], t0), n1 = fmaxf(m[1], t1);
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
                n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, o));
                n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, o));
            }
            const float f0 = n0 == m[0] ? 1.f : ex2(m[0] - n0), f1 = n1 == m[1] ? 1.f : ex2(m[1] - n1);
            m[0] = n0; m[1] = n1;
            l[0] *= f0; l[1] *= f1;
#pragma unroll
            for (int t = 0; t < HD / 16; ++t) { acc[t][0] *= f0; acc[t][1] *= f1; acc[t][2] *= f0; acc[t][3] *= f1; }
        }
        const float r0 = m[0] == -INFINITY ? 0.f : m[0], r1 = m[1] == -INFINITY ? 0.f : m[1];      // (nothing seen yet)
        s[0] = ex2(s[0] - r0); s[1] = ex2(s[1] - r1); s[2] = ex2(s[2] - r0); s[3] = ex2(s[3] - r1);
        l[0] += s[0] + s[2];
        l[1] += s[1] + s[3];
        page_values<KVT, HD, S::PP, PAIR>(f, s, acc);
    }
    src.end();
    if constexpr (PAIR) {                                    // both bands together
        const float f = 1.f / ((j & 2 ? kPairLow : kPairUp) * kCodeScale);
#pragma unroll
        for (int t = 0; t < HD / 16; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                acc[t][e] *= f;
                acc[t][e] += __shfl_xor_sync(0xffffffffu, acc[t][e], 2);
            }
    }
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
        l[0] += __shfl_xor_sync(0xffffffffu, l[0], o);
        l[1] += __shfl_xor_sync(0xffffffffu, l[1], o);
    }
}

template <typename KVT, typename RT, int HD>
__device__ __forceinline__ void walk_pages(const AttnPagedParams& p, const Block& k, const PagedSpan& span, int v, int v1, int step, PageSource<KVT, HD>& src,
                                           const uint2* qf, const float* qscale, float (&acc)[HD / 16][4], float (&m)[2], float (&l)[2]) {
    using S = SplitShape<KVT, RT, HD>;
    if constexpr (S::MAY_PAIR)
        if (S::pair(k.count)) return walk_rows<KVT, RT, HD, true>(p, k, span, v, v1, step, src, qf, qscale, acc, m, l);
    walk_rows<KVT, RT, HD, false>(p, k, span, v, v1, step, src, qf, qscale, acc, m, l);
}

// Shared memory of a CTA's rings, and of its warps' results, which lie over them
template <typename KVT, int HD, int TEAM>
__host__ __device__ constexpr int split_ring_bytes() {
    constexpr int rings = kSplitWarps * PageSource<KVT, HD>::kRing, results = TEAM > 1 ? kSplitWarps * split_part_floats(HD) * 4 : 0;
    return rings > results ? rings : results;
}

// Row i of a block: its row of the call's tensors, head, and position
__device__ __forceinline__ void block_row(const AttnPagedParams& p, const Block& k, int i, int& row, int& h, int& pos) {
    const int r = k.first + i, t = r / p.group;
    row = k.s.r0 + t;
    h = k.kvh * p.group + r % p.group;
    pos = k.s.len - k.s.n + t;
}

// Result of dims d, d + 1 of a row: sums over the total. True if it is not finite (a row that sees nothing is 0).
template <typename KVT, typename RT, int HD>
__device__ __forceinline__ bool put_pair(const AttnPagedParams& p, int row, int h, int pos, int d, float x, float y, float l) {
    const float inv = pos < 0 ? 0.f : p.c.v_scale * (sizeof(KVT) == 1 ? kCodeScale : 1.f) / l;
    x = pos < 0 ? 0.f : x * inv;
    y = pos < 0 ? 0.f : y * inv;
    const size_t at = (size_t)row * p.heads * HD + (size_t)h * HD + d;
    const bool odd = !(fabsf(x) <= 3.4e38f) || !(fabsf(y) <= 3.4e38f);
    if (p.gate && pos >= 0) { x *= p.gate[at]; y *= p.gate[at + 1]; }      // (of a padding row it may hold anything)
    RT* o = static_cast<RT*>(p.out) + (size_t)row * p.out_stride + (size_t)h * HD + d;
    if (reinterpret_cast<uintptr_t>(o) % (2 * sizeof(RT)) == 0) {
        if constexpr (sizeof(RT) == 2) *reinterpret_cast<uint32_t*>(o) = f32x2_to_bf16(x, y);
        else *reinterpret_cast<float2*>(o) = make_float2(x, y);
    } else {
        Elem<RT>::put(o, 0, x);
        Elem<RT>::put(o, 1, y);
    }
    return odd;
}

// ---- the positions of all sequences dealt out evenly ---------------------------------------------------------------------
// Page counts of a batch's sequences differ, and so does how many sequences there are for 148 SMs: so the pages of all (sequence, K/V
// head, block of rows) are laid end to end and cut into as many equal shares as there are teams (a CTA's warps together, or each warp alone),
// and the shares' partial results of an item that a cut goes through are put together by attn_join_kernel. Bound by HBM with many bf16 pages: 64 sequences in
// a window of 4096, 32 / 8 heads of 128, 167 us for 932 MB, 85 % of the measured copy rate. By the instructions that widen the codes with 4-bit
// pages: 128 sequences of up to 8000 positions, the same heads, 144 us for 602 MB, 64 %. By latency (lengths, queries, page ids, pages, the
// CTA's results, the join: some 1 to 2 us each) with few: one user in a window of 1024, 10 us. Sequences of more than
// kSplitRows (token, head) pairs are left to the kernels for prompts.
// (sequences, pages of their items before them) -> plan in shared memory; returns the total
__device__ __forceinline__ int split_blocks(const AttnPagedParams& p, int n) {
    const long long rows = (long long)n * p.group;
    return rows > kSplitRows ? 0 : (int)((rows + 7) / 8);
}

// The total cut into equal shares, the first `more` of them one larger
struct Shares {
    unsigned long long each;
    unsigned teams, more;
    __device__ __forceinline__ static unsigned long long div(unsigned long long a, unsigned long long b) {
        return (a | b) >> 32 ? a / b : (unsigned)a / (unsigned)b;
    }
    __device__ __forceinline__ Shares(unsigned long long total, int max_teams, int least) {
        const unsigned long long n = div(total, (unsigned)least);
        teams = n < 1 ? 1u : n < (unsigned)max_teams ? (unsigned)n : (unsigned)max_teams;
        each = div(total, teams);
        more = (unsigned)(total - each * teams);
    }
    // of `size` each, of a total that is so many of them
    __device__ __forceinline__ Shares(unsigned long long total, unsigned size) : each(size), teams((unsigned)div(total, size)), more(0) {}
    __device__ __forceinline__ unsigned long long start(unsigned t) const { return each * t + min(t, more); }
    __device__ __forceinline__ unsigned holder(unsigned long long x) const {         // of x < total
        const unsigned long long big = (each + 1) * more;
        return x < big ? (unsigned)div(x, each + 1) : more + (unsigned)div(x - big, each);
    }
};

// Units of an item in the plan: pages and what p.item_cost adds; with few items (`size` > 0) pages up to a multiple of the shares' size, so that no
// share has parts of two items (that one ended 5 us after the others).
__device__ __forceinline__ unsigned item_units(const AttnPagedParams& p, unsigned size, int pages) {
    const unsigned n = (unsigned)max(1, pages + p.item_cost);
    return size > 0 ? (n + size - 1) / size * size : n;
}
// The size of a share, 0 where items are many: with at most one share more for every item there are no more than p.max_teams. Called by all of a
// CTA's threads; a sequence for each of them, since there are fewer than p.max_teams / 4 items.
template <int TEAM>
__device__ __forceinline__ unsigned share_size(const AttnPagedParams& p, unsigned long long (&sums)[2][kSplitWarps]) {
    if (p.item_cost > 0) return 0;
    unsigned long long n = 0, items = 0;
    if ((int)threadIdx.x < p.r.batch) {
        const PagedSeq s = paged_seq(p.r, p.c.pt_stride, threadIdx.x, false);
        items = (unsigned long long)split_blocks(p, s.n) * p.c.kv_heads;
        if (items > 0) n = item_units(p, 0, paged_span(p, s.len - s.n, s.len - 1).count) * items;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        n += __shfl_xor_sync(0xffffffffu, n, o);
        items += __shfl_xor_sync(0xffffffffu, items, o);
    }
    if (threadIdx.x % 32 == 0) { sums[0][threadIdx.x / 32] = n; sums[1][threadIdx.x / 32] = items; }
    __syncthreads();
    n = items = 0;
#pragma unroll
    for (int w = 0; w < kSplitWarps; ++w) { n += sums[0][w]; items += sums[1][w]; }
    __syncthreads();
    const unsigned teams = (unsigned)p.max_teams - (unsigned)items;
    return max((unsigned)TEAM, (unsigned)Shares::div(n + teams - 1, teams));
}

// TEAM: warps of a team, 1 or kSplitWarps
template <typename KVT, typename RT, int HD, int TEAM>
__global__ void __launch_bounds__(32 * kSplitWarps, 2) attn_split_kernel(const __grid_constant__ AttnPagedParams p) {
    using S = SplitShape<KVT, RT, HD>;
    extern __shared__ __align__(16) unsigned char sm[];
    uint2* qf_all = reinterpret_cast<uint2*>(sm);                                        // [warp][QWORDS]
    unsigned char* ring = sm + (size_t)kSplitWarps * S::QWORDS * 8;
    float* red = reinterpret_cast<float*>(ring);                                         // TEAM > 1: [warp][8][W], a row's maximum and total behind its sums
    unsigned long long* plan = reinterpret_cast<unsigned long long*>(ring + split_ring_bytes<KVT, HD, TEAM>());      // [batch + 1]
    __shared__ float qs_all[kSplitWarps][8];
    __shared__ unsigned long long warp_sum_[kSplitWarps], sums[2][kSplitWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, j = lane & 3;
    pdl_launch_dependents();
    const unsigned size = share_size<TEAM>(p, sums);
    // units before each sequence
    unsigned long long before = 0;
    for (int b0 = 0; b0 < p.r.batch; b0 += 32 * kSplitWarps) {
        const int b = b0 + tid;
        unsigned long long n = 0;
        if (b < p.r.batch) {
            const PagedSeq s = paged_seq(p.r, p.c.pt_stride, b, blockIdx.x == 0);
            const int blocks = split_blocks(p, s.n);
            if (blocks > 0) n = (unsigned long long)item_units(p, size, paged_span(p, s.len - s.n, s.len - 1).count) * blocks * p.c.kv_heads;
        }
        unsigned long long x = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) warp_sum_[warp] = x;
        __syncthreads();
        unsigned long long all = 0, mine = 0;
#pragma unroll
        for (int w = 0; w < kSplitWarps; ++w) {
            if (w < warp) mine += warp_sum_[w];
            all += warp_sum_[w];
        }
        if (b < p.r.batch) plan[b] = before + mine + x - n;
        before += all;
        __syncthreads();
    }
    if (tid == 0) plan[p.r.batch] = before;
    __syncthreads();
    if (blockIdx.x == 0)
        for (int b = tid; b <= p.r.batch; b += 32 * kSplitWarps) p.plan[b] = plan[b];
    const unsigned long long total = before;
    if (total == 0) return;
    const Shares shares = size > 0 ? Shares(total, size) : Shares(total, p.max_teams, TEAM + p.item_cost);
    const unsigned team = TEAM == 1 ? blockIdx.x * kSplitWarps + warp : blockIdx.x;
    if (team >= shares.teams) return;
    const unsigned long long start = shares.start(team), end = shares.start(team + 1);
    int b = 0, hi = p.r.batch;
    while (hi - b > 1) {
        const int mid = (b + hi) / 2;
        if (plan[mid] <= start) b = mid; else hi = mid;
    }
    const uint2* qf = qf_all + warp * S::QWORDS;
    const float* qscale = qs_all[warp];
    unsigned long long at = start;
    while (at < end) {
        while (plan[b + 1] <= at) ++b;
        Block k;
        k.b = b;
        k.s = paged_seq(p.r, p.c.pt_stride, b, false);
        const int blocks = split_blocks(p, k.s.n);
        const PagedSpan span = paged_span(p, k.s.len - k.s.n, k.s.len - 1);
        const unsigned count = item_units(p, size, span.count);
        const unsigned long long rest = at - plan[b], left = end - at, item64 = Shares::div(rest, count);
        const unsigned c0 = (unsigned)(rest - item64 * count), c1 = left < count - c0 ? c0 + (unsigned)left : count, item = (unsigned)item64;
        const int v0 = max(0, (int)c0 - p.item_cost), v1 = max(0, (int)c1 - p.item_cost);      // pages
        k.kvh = (int)(item / (unsigned)blocks);
        k.first = (int)(item % (unsigned)blocks) * 8;
        k.count = min(8, k.s.n * p.group - k.first);
        const int mine0 = v0 + (TEAM > 1 ? warp : 0);
        PageSource<KVT, HD> page(p, k, span, mine0, min(v1, span.count), TEAM, ring + warp * PageSource<KVT, HD>::kRing);
        __syncwarp();
        pack_queries<RT, S::QP, HD, typename S::F>(p, k, S::pair(k.count), const_cast<uint2*>(qf), const_cast<float*>(qscale), lane);
        __syncwarp();
        float acc[HD / 16][4], m[2], l[2];
        walk_pages<KVT, RT, HD>(p, k, span, mine0, min(v1, span.count), TEAM, page, qf, qscale, acc, m, l);
        const bool whole = c0 == 0 && c1 == count;
        float* part = p.part + ((size_t)team * 2 + (at == start ? 0 : 1)) * S::PART;
        if constexpr (TEAM == 1) {
            bool odd = false;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int i = 2 * j + c;
                if (i >= k.count) continue;
                if (whole) {
                    int row, h, pos;
                    block_row(p, k, i, row, h, pos);
#pragma unroll
                    for (int t = 0; t < HD / 16; ++t) odd |= put_pair<KVT, RT, HD>(p, row, h, pos, S::F::vdim(t, g), acc[t][c], acc[t][2 + c], l[c]);
                } else {
#pragma unroll
                    for (int t = 0; t < HD / 16; ++t) *reinterpret_cast<float2*>(part + i * S::W + S::F::vdim(t, g)) = make_float2(acc[t][c], acc[t][2 + c]);
                    if (g == 0) { part[i * S::W + HD] = m[c]; part[i * S::W + HD + 1] = l[c]; }
                }
            }
            if (__any_sync(0xffffffffu, odd)) {
                for (int i = 0; i < k.count; ++i) {
                    int row, h, pos;
                    block_row(p, k, i, row, h, pos);
                    careful_row<KVT, RT, HD>(p, k.b, pos, row, h);
                }
            }
        } else {
            if (PageSource<KVT, HD>::kRing > 0) __syncthreads();         // the rings have been read
            float* mine = red + warp * S::PART;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int i = 2 * j + c;
#pragma unroll
                for (int t = 0; t < HD / 16; ++t) *reinterpret_cast<float2*>(mine + i * S::W + S::F::vdim(t, g)) = make_float2(acc[t][c], acc[t][2 + c]);
                if (g == 0) { mine[i * S::W + HD] = m[c]; mine[i * S::W + HD + 1] = l[c]; }
            }
            __syncthreads();
            // a warp per row: the team's warps' results together
            bool odd = false;
            const int i = warp;
            if (i < k.count) {
                float mx = -INFINITY, lt = 0.f;
#pragma unroll
                for (int w = 0; w < kSplitWarps; ++w) mx = fmaxf(mx, red[w * S::PART + i * S::W + HD]);
                const float ref = mx == -INFINITY ? 0.f : mx;
                float2 o[HD / 64];
#pragma unroll
                for (int e = 0; e < HD / 64; ++e) o[e] = make_float2(0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kSplitWarps; ++w) {
                    const float* r = red + w * S::PART + i * S::W;
                    const float f = ex2(r[HD] - ref);
                    lt = fmaf(r[HD + 1], f, lt);
#pragma unroll
                    for (int e = 0; e < HD / 64; ++e) {
                        const float2 x = *reinterpret_cast<const float2*>(r + e * 64 + lane * 2);
                        o[e].x = fmaf(x.x, f, o[e].x);
                        o[e].y = fmaf(x.y, f, o[e].y);
                    }
                }
                int row, h, pos;
                block_row(p, k, i, row, h, pos);
#pragma unroll
                for (int e = 0; e < HD / 64; ++e) {
                    if (whole) odd |= put_pair<KVT, RT, HD>(p, row, h, pos, e * 64 + lane * 2, o[e].x, o[e].y, lt);
                    else *reinterpret_cast<float2*>(part + i * S::W + e * 64 + lane * 2) = o[e];
                }
                if (!whole && lane == 0) { part[i * S::W + HD] = mx; part[i * S::W + HD + 1] = lt; }
                if (__any_sync(0xffffffffu, odd)) careful_row<KVT, RT, HD>(p, k.b, pos, row, h);
            }
            __syncthreads();
        }
        at += c1 - c0;
    }
}

// Joins the partial results of the items that a share's end goes through: `WPR` warps per row, a CTA for kSplitWarps / WPR rows of an item.
template <typename KVT, typename RT, int HD, int TEAM>
__global__ void __launch_bounds__(32 * kSplitWarps) attn_join_kernel(const __grid_constant__ AttnPagedParams p, int max_blocks) {
    using S = SplitShape<KVT, RT, HD>;
    constexpr int WPR = TEAM == 1 ? 1 : kSplitWarps;
    __shared__ float red[kSplitWarps][HD + 2];
    __shared__ unsigned long long sums[2][kSplitWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per = max_blocks * p.c.kv_heads, b = (int)blockIdx.x / per, item = (int)blockIdx.x % per;
    const int i = WPR == 1 ? warp : (int)blockIdx.y;
    pdl_launch_dependents();
    // Where the item lies in the plan, while the other kernel is at work: worked out again where a thread has one sequence at most, else read
    const unsigned size = share_size<TEAM>(p, sums);
    unsigned long long total = 0, o0 = 0;
    const bool own_plan = p.r.batch <= 32 * kSplitWarps;
    if (own_plan) {
        unsigned long long n = 0;
        if ((int)threadIdx.x < p.r.batch) {
            const PagedSeq s = paged_seq(p.r, p.c.pt_stride, threadIdx.x, false);
            const int blocks = split_blocks(p, s.n);
            if (blocks > 0) n = (unsigned long long)item_units(p, size, paged_span(p, s.len - s.n, s.len - 1).count) * blocks * p.c.kv_heads;
        }
        unsigned long long before = (int)threadIdx.x < b ? n : 0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            n += __shfl_xor_sync(0xffffffffu, n, o);
            before += __shfl_xor_sync(0xffffffffu, before, o);
        }
        if (lane == 0) { sums[0][warp] = n; sums[1][warp] = before; }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kSplitWarps; ++w) { total += sums[0][w]; o0 += sums[1][w]; }
    }
    Block k;
    k.b = b;
    k.s = paged_seq(p.r, p.c.pt_stride, b, false);
    const int blocks = split_blocks(p, k.s.n);
    if (!own_plan) {
        pdl_wait();
        total = __ldcg(p.plan + p.r.batch);
        o0 = __ldcg(p.plan + b);
    }
    const bool mine = item < blocks * p.c.kv_heads;
    k.kvh = mine ? item / blocks : 0;
    k.first = mine ? item % blocks * 8 : 0;
    k.count = mine ? min(8, k.s.n * p.group - k.first) : 0;
    if (i >= k.count) {
        if (own_plan) pdl_wait();
        return;
    }
    const unsigned count = item_units(p, size, paged_span(p, k.s.len - k.s.n, k.s.len - 1).count);
    o0 += (unsigned long long)item * count;
    const Shares shares = size > 0 ? Shares(total, size) : Shares(total, p.max_teams, TEAM + p.item_cost);
    const unsigned t0 = shares.holder(o0), t1 = shares.holder(o0 + count - 1), slot0 = shares.start(t0) == o0 ? 0 : 1;
    if (own_plan) pdl_wait();
    if (t0 == t1) return;                        // one team held it all and wrote the result
    // partial results, four at a time: maximum so far, total and sums
    float mx = -INFINITY, lt = 0.f;
    float2 o[HD / 64];
#pragma unroll
    for (int e = 0; e < HD / 64; ++e) o[e] = make_float2(0.f, 0.f);
    for (unsigned t = t0 + (WPR == 1 ? 0 : warp); t <= t1; t += 4 * WPR) {
        float pm[4], pl[4];
        float2 x[4][HD / 64];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const unsigned tu = t + u * WPR;
            pm[u] = -INFINITY;
            pl[u] = 0.f;
            const float* r = p.part + ((size_t)tu * 2 + (tu == t0 ? slot0 : 0)) * S::PART + i * S::W;
#pragma unroll
            for (int e = 0; e < HD / 64; ++e) x[u][e] = tu <= t1 ? __ldcg(reinterpret_cast<const float2*>(r + e * 64 + lane * 2)) : make_float2(0.f, 0.f);
            if (tu <= t1) {
                const float2 ml = __ldcg(reinterpret_cast<const float2*>(r + HD));
                pm[u] = ml.x;
                pl[u] = ml.y;
            }
        }
        const float mn = fmaxf(fmaxf(mx, fmaxf(pm[0], pm[1])), fmaxf(pm[2], pm[3])), ref = mn == -INFINITY ? 0.f : mn, f = ex2(mx - ref);
        mx = mn;
        lt *= f;
#pragma unroll
        for (int e = 0; e < HD / 64; ++e) { o[e].x *= f; o[e].y *= f; }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float fu = ex2(pm[u] - ref);
            lt = fmaf(pl[u], fu, lt);
#pragma unroll
            for (int e = 0; e < HD / 64; ++e) {
                o[e].x = fmaf(x[u][e].x, fu, o[e].x);
                o[e].y = fmaf(x[u][e].y, fu, o[e].y);
            }
        }
    }
    if constexpr (WPR > 1) {
#pragma unroll
        for (int e = 0; e < HD / 64; ++e) *reinterpret_cast<float2*>(&red[warp][e * 64 + lane * 2]) = o[e];
        if (lane == 0) { red[warp][HD] = mx; red[warp][HD + 1] = lt; }
        __syncthreads();
        if (warp > 0) return;
#pragma unroll
        for (int w = 0; w < WPR; ++w) mx = fmaxf(mx, red[w][HD]);
        const float ref = mx == -INFINITY ? 0.f : mx;
        lt = 0.f;
#pragma unroll
        for (int e = 0; e < HD / 64; ++e) o[e] = make_float2(0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WPR; ++w) {
            const float f = ex2(red[w][HD] - ref);
            lt = fmaf(red[w][HD + 1], f, lt);
#pragma unroll
            for (int e = 0; e < HD / 64; ++e) {
                o[e].x = fmaf(red[w][e * 64 + lane * 2], f, o[e].x);
                o[e].y = fmaf(red[w][e * 64 + lane * 2 + 1], f, o[e].y);
            }
        }
    }
    int row, h, pos;
    block_row(p, k, i, row, h, pos);
    bool odd = false;
#pragma unroll
    for (int e = 0; e < HD / 64; ++e) odd |= put_pair<KVT, RT, HD>(p, row, h, pos, e * 64 + lane * 2, o[e].x, o[e].y, lt);
    if (__any_sync(0xffffffffu, odd)) careful_row<KVT, RT, HD>(p, k.b, pos, row, h);
}

// ---- more rows: a CTA per block of eight rows of a K/V head, its warps through the pages in turn ------------------------------
template <typename KVT, typename RT, int HD>
__global__ void __launch_bounds__(32 * kSplitWarps, 2) attn_blocks_kernel(const __grid_constant__ AttnPagedParams p) {
    using S = SplitShape<KVT, RT, HD>;
    extern __shared__ __align__(16) unsigned char sm[];
    uint2* qf = reinterpret_cast<uint2*>(sm);
    unsigned char* ring = sm + (size_t)S::QWORDS * 8;
    float* red = reinterpret_cast<float*>(ring);
    __shared__ float qscale[8];
    __shared__ int found[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, j = lane & 3;
    // which sequence's block this is: blocks of those with more than kSplitRows rows, the last sequence and its later rows (which see more) first
    if (warp == 0) {
        int want = (int)(gridDim.x - 1 - blockIdx.x), at = -1;
        for (int b0 = 0; b0 < p.r.batch && at < 0; b0 += 32) {
            const int b = b0 + lane;
            int n = 0;
            if (b < p.r.batch) {
                const PagedSeq s = paged_seq(p.r, p.c.pt_stride, b, blockIdx.x == 0 && blockIdx.y == 0);
                const long long rows = (long long)s.n * p.group;
                n = rows > kSplitRows ? (int)((rows + 7) / 8) : 0;
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
                const int before = __shfl_sync(0xffffffffu, x - n, src);
                at = b0 + src;
                want -= before;
            } else {
                want -= __shfl_sync(0xffffffffu, x, 31);
            }
        }
        if (lane == 0) { found[0] = at; found[1] = want; }
    }
    __syncthreads();
    if (found[0] < 0) return;
    Block k;
    k.b = found[0];
    k.s = paged_seq(p.r, p.c.pt_stride, k.b, false);
    k.kvh = blockIdx.y;
    k.first = found[1] * 8;
    k.count = min(8, k.s.n * p.group - k.first);
    const int pos0 = k.s.len - k.s.n;
    const PagedSpan span = paged_span(p, pos0 + k.first / p.group, pos0 + (k.first + k.count - 1) / p.group);
    PageSource<KVT, HD> page(p, k, span, warp, span.count, kSplitWarps, ring + warp * PageSource<KVT, HD>::kRing);
    if (warp == 0) pack_queries<RT, S::QP, HD, typename S::F>(p, k, S::pair(k.count), qf, qscale, lane);
    __syncthreads();
    float acc[HD / 16][4], m[2], l[2];
    walk_pages<KVT, RT, HD>(p, k, span, warp, span.count, kSplitWarps, page, qf, qscale, acc, m, l);
    if (PageSource<KVT, HD>::kRing > 0) __syncthreads();                 // the rings have been read
    float* mine = red + warp * S::PART;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const int i = 2 * j + c;
#pragma unroll
        for (int t = 0; t < HD / 16; ++t) *reinterpret_cast<float2*>(mine + i * S::W + S::F::vdim(t, g)) = make_float2(acc[t][c], acc[t][2 + c]);
        if (g == 0) { mine[i * S::W + HD] = m[c]; mine[i * S::W + HD + 1] = l[c]; }
    }
    __syncthreads();
    const int i = warp;
    if (i >= k.count) return;
    float mx = -INFINITY, lt = 0.f;
#pragma unroll
    for (int w = 0; w < kSplitWarps; ++w) mx = fmaxf(mx, red[w * S::PART + i * S::W + HD]);
    const float ref = mx == -INFINITY ? 0.f : mx;
    float2 o[HD / 64];
#pragma unroll
    for (int e = 0; e < HD / 64; ++e) o[e] = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kSplitWarps; ++w) {
        const float* r = red + w * S::PART + i * S::W;
        const float f = ex2(r[HD] - ref);
        lt = fmaf(r[HD + 1], f, lt);
#pragma unroll
        for (int e = 0; e < HD / 64; ++e) {
            const float2 x = *reinterpret_cast<const float2*>(r + e * 64 + lane * 2);
            o[e].x = fmaf(x.x, f, o[e].x);
            o[e].y = fmaf(x.y, f, o[e].y);
        }
    }
    int row, h, pos;
    block_row(p, k, i, row, h, pos);
    bool odd = false;
#pragma unroll
    for (int e = 0; e < HD / 64; ++e) odd |= put_pair<KVT, RT, HD>(p, row, h, pos, e * 64 + lane * 2, o[e].x, o[e].y, lt);
    if (__any_sync(0xffffffffu, odd)) careful_row<KVT, RT, HD>(p, k.b, pos, row, h);
}

template <typename KVT, typename RT, int HD, int TEAM>
cudaError_t split_launch(AttnPagedParams p, int sm_count, cudaStream_t st) {
    using S = SplitShape<KVT, RT, HD>;
    const size_t smem = (size_t)kSplitWarps * S::QWORDS * 8 + split_ring_bytes<KVT, HD, TEAM>() + ((size_t)p.r.batch + 1) * 8;
    cudaError_t e = cudaFuncSetAttribute(attn_split_kernel<KVT, RT, HD, TEAM>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
    if (e != cudaSuccess) return e;
    const int ctas = 2 * sm_count;
    p.max_teams = TEAM == 1 ? ctas * kSplitWarps : ctas;
    // Beside its pages an item costs what comes before and after them, measured in pages: 7 small ones of 4 bits for a warp alone (2: 170 us for 128
    // sequences of up to 8000 positions with weights in bf16, 4: 165, 6: 160, 8: 161; 256 short ones 68, 57, 52, 52), 4 others (2: 86 us for 200 sequences of up to 2000, 4:
    // 81, 8: 84), and two for each warp of a team (1: 172 us for 64 sequences in a window of 4096, 2: 164, 4: 166). Where a share has parts of two items at
    // most, that is the same for all and left out.
    p.item_cost = (long long)p.r.batch * p.c.kv_heads * 4 < p.max_teams ? 0 : TEAM > 1 ? 2 * TEAM : sizeof(KVT) == 1 ? 7 : 4;
    attn_split_kernel<KVT, RT, HD, TEAM><<<ctas, 32 * kSplitWarps, smem, st>>>(p);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    const int blocks = p.r.row_start ? kSplitRows / 8 : 1;
    const int rows = p.r.row_start ? 8 : std::min(8, p.group);
    return launch_after(attn_join_kernel<KVT, RT, HD, TEAM>, dim3(p.r.batch * p.c.kv_heads * blocks, TEAM == 1 ? 1 : rows), 32 * kSplitWarps, 0, st, p, blocks);
}

template <typename KVT, typename RT, int HD>
cudaError_t launch_one(const AttnPagedParams& p, int sm_count, cudaStream_t st) {
    using S = SplitShape<KVT, RT, HD>;
    // Each warp alone where there are sequences and heads enough to give most of them whole items: nothing to put together in a CTA. A warp / a CTA a share,
    // in us, 8 K/V heads, sequences of up to 3000 positions: bf16 pages, heads of 128, 464 items 78 / 77, 600 93 / 105, 1024 147 / 160, 2048 280 / 305;
    // heads of 64 38 / 42, 46 / 55, 73 / 86, 134 / 162; fp32 pages, heads of 128, 224 / 225, 264 / 298, 437 / 489, 862 / 979; 4-bit pages, fp32 rows, heads
    // of 128, 51 / 60, 58 / 81, 89 / 123, 168 / 233. Of up to 300 positions the warp is ahead by more (bf16, 128, 600 items: 27 / 38). So over
    // 4-bit pages it would be from about 300 items on; one rule for all stays behind there.
    const long long items = (long long)p.r.batch * p.c.kv_heads;
    const bool prompts = paged_prompts(p.r.row_start, p.r.rows, p.r.max_rows, p.group);
    constexpr bool TILES = sizeof(KVT) <= 2 && sizeof(RT) == 2;
    constexpr int dtype = sizeof(KVT) == 1 ? MLB_DT_FP4_E2M1 : MLB_DT_BF16;
    PromptMaps maps;
    cudaError_t e = TILES && prompts ? attn_prompt_maps(p, dtype, HD, &maps) : cudaSuccess;
    if (e != cudaSuccess) return e;
    e = items >= 4LL * sm_count ? split_launch<KVT, RT, HD, 1>(p, sm_count, st) : split_launch<KVT, RT, HD, kSplitWarps>(p, sm_count, st);
    if (e != cudaSuccess || !prompts) return e;
    if constexpr (TILES) {
        return attn_prompt_launch(p, dtype, HD, maps, st);
    } else {
        const size_t smem = (size_t)S::QWORDS * 8 + split_ring_bytes<KVT, HD, kSplitWarps>();
        e = cudaFuncSetAttribute(attn_blocks_kernel<KVT, RT, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, 100 * 1024);
        if (e != cudaSuccess) return e;
        const long long blocks = (long long)p.r.rows * p.group / 8 + p.r.batch;
        attn_blocks_kernel<KVT, RT, HD><<<dim3((unsigned)blocks, p.c.kv_heads), 32 * kSplitWarps, smem, st>>>(p);
        return cudaGetLastError();
    }
}

template <typename KVT, typename RT>
cudaError_t launch_types(const AttnPagedParams& p, int hd, int sm_count, cudaStream_t st) {
    return hd == 64 ? launch_one<KVT, RT, 64>(p, sm_count, st) : launch_one<KVT, RT, 128>(p, sm_count, st);
}

}  // namespace

size_t attn_paged_part_bytes(int sm_count) { return (size_t)sm_count * 2 * kSplitWarps * 2 * split_part_floats(128) * 4; }

cudaError_t attn_paged_launch(const AttnPagedParams& p, int dtype, int row_dtype, int head_dim, int sm_count, cudaStream_t st) {
    const bool f = row_dtype == MLB_DT_F32;
    if (dtype == MLB_DT_F32) return f ? launch_types<float, float>(p, head_dim, sm_count, st) : launch_types<float, bf16_t>(p, head_dim, sm_count, st);
    if (dtype == MLB_DT_BF16) return f ? launch_types<bf16_t, float>(p, head_dim, sm_count, st) : launch_types<bf16_t, bf16_t>(p, head_dim, sm_count, st);
    return f ? launch_types<fp4_t, float>(p, head_dim, sm_count, st) : launch_types<fp4_t, bf16_t>(p, head_dim, sm_count, st);
}

}  // namespace mlb
