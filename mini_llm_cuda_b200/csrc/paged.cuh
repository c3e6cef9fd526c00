// Shared pieces of the operators over a caller's paged K/V cache (mlb_paged_kv, mlb_new_rows): what the kernels get, how they read the
// caller's row ranges and page tables without trusting them, and the 4-bit format.
#pragma once
#include <cuda_fp16.h>

#include <cstdint>

#include "../../include/mlb.h"
#include "kernels.cuh"

namespace mlb {

struct fp4_t { unsigned char b; };      // two e2m1 codes; tag of a 4-bit cache

// What a kernel found wrong with the caller's data (mlb_ops_status)
enum PagedErr : int { PG_ROWS = 1, PG_MAX_ROWS = 2, PG_LONG = 3, PG_PAGE = 4, PG_ROPE = 5, PG_WAIT = 6 };

struct PagedCache {
    void *kpool, *vpool;
    unsigned char *kscale, *vscale;
    const int* page_table;
    int pt_stride, num_pages, kv_heads;
    float k_scale, v_scale;
};

struct PagedRows {
    const int* row_start;       // or null: sequence b brings row b
    const int* kv_lens;
    int batch, rows, max_rows;
    int* err;
};

struct PagedSeq {
    int r0, n, len;             // first row, rows, cached positions with them; n = 0 where the caller's data cannot be used
};

__device__ __forceinline__ PagedSeq paged_seq(const PagedRows& p, int pt_stride, int b, bool report) {
    PagedSeq s;
    s.len = max(0, p.kv_lens[b]);                // (on its way together with the others)
    if (p.row_start) {
        s.r0 = p.row_start[b];
        const int r1 = p.row_start[b + 1];
        s.n = r1 - s.r0;
        if (s.r0 < 0 || r1 < s.r0 || r1 > p.rows) {
            if (report) atomicExch(p.err, PG_ROWS);
            s.r0 = s.n = 0;
        } else if (p.max_rows > 0 && s.n > p.max_rows) {
            if (report) atomicExch(p.err, PG_MAX_ROWS);
            s.n = 0;
        }
    } else {
        s.r0 = b;
        s.n = b < p.rows ? 1 : 0;
    }
    if (s.n > 0 && s.len > (long long)pt_stride * kKvBlock) {
        if (report) atomicExch(p.err, PG_LONG);
        s.n = 0;
    }
    return s;
}

// Page `i` of sequence b; a bad id reads as page 0, or -1 for a writer.
__device__ __forceinline__ int paged_page(const PagedCache& c, int* err, int b, int i, int bad) {
    int id = c.page_table[(size_t)b * c.pt_stride + i];
    if ((unsigned)id >= (unsigned)c.num_pages) {
        atomicExch(err, PG_PAGE);
        id = bad;
    }
    return id;
}

__device__ __forceinline__ float f16_lo(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)(w & 0xffffu))); }
__device__ __forceinline__ float f16_hi(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)(w >> 16))); }
__device__ __forceinline__ uint32_t f32x2_to_bf16(float lo, float hi) {
    uint32_t o;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(o) : "f"(hi), "f"(lo));
    return o;
}
__device__ __forceinline__ uint32_t f32x2_to_f16(float lo, float hi) {
    uint32_t o;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(o) : "f"(hi), "f"(lo));
    return o;
}

// Two e2m1 codes of a byte -> two halves (exact), low code first; four bytes at once
__device__ __forceinline__ void e2m1x8_to_f16(uint32_t codes, uint32_t (&o)[4]) {
    asm("{\n"
        ".reg .b8 b0, b1, b2, b3;\n"
        "mov.b32 {b0, b1, b2, b3}, %4;\n"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n"
        "}\n"
        : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3])
        : "r"(codes));
}
// Low four bits of `code`; its exponent and mantissa at the low end of a float's exponent are the value times 2^-126
__device__ __forceinline__ float e2m1_value(uint32_t code) { return __uint_as_float((code & 8u) << 28 | (code & 7u) << 22) * 8.507059173023462e37f; }
// Two e4m3 values -> two halves (exact)
__device__ __forceinline__ uint32_t e4m3x2_to_f16(uint32_t two) {
    uint32_t o;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(o) : "h"((unsigned short)two));
    return o;
}
__device__ __forceinline__ float e4m3_to_f32(unsigned char x) {
    const uint32_t h = e4m3x2_to_f16(x);
    return __half2float(__ushort_as_half((unsigned short)(h & 0xffffu)));
}
__device__ __forceinline__ unsigned char f32_to_e4m3(float x) {      // nearest, ties to even, at most 448
    unsigned short o;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(o) : "f"(0.f), "f"(x));
    return (unsigned char)(o & 0xff);
}
// Eight fp32 values -> eight e2m1 codes (nearest, ties to the even code, at most 6)
__device__ __forceinline__ uint32_t f32x8_to_e2m1(const float (&x)[8]) {
    uint32_t o;
    asm("{\n"
        ".reg .b8 b0, b1, b2, b3;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n"
        "mov.b32 %0, {b0, b1, b2, b3};\n"
        "}\n"
        : "=r"(o)
        : "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]));
    return o;
}

struct AttnPagedParams {
    PagedCache c;
    PagedRows r;
    const void* q; long long q_stride;
    const float* gate;
    void* out; long long out_stride;
    int heads, group;           // query heads, and per K/V head
    uint32_t group_inv;         // 2^32 / group + 1, of more than one
    float scale;                // of the scores
    int window, sinks;
    float* part;                // partial results, paged_part_floats() each
    unsigned long long* plan;   // [batch + 1] pages before a sequence, as the splitting kernel laid them out
    int max_teams, item_cost;   // of the splitting kernel
};

// Pages that a block of rows sees: `sink_pages` from the first one on, then those from `first` on; `count` in all.
struct PagedSpan {
    int sink_pages, first, count;
    __device__ __forceinline__ int page(int v) const { return v < sink_pages ? v : first + (v - sink_pages); }
};
// pa, pb: positions of the block's first and last row
__device__ __forceinline__ PagedSpan paged_span(const AttnPagedParams& p, int pa, int pb) {
    PagedSpan s;
    if (pb < 0) {
        s.sink_pages = s.first = s.count = 0;
        return s;
    }
    const int low = p.window > 0 ? max(0, max(pa, 0) - p.window + 1) : 0;
    s.first = low / kKvBlock;
    s.sink_pages = p.window > 0 && p.sinks > 0 ? min((min(p.sinks, pb + 1) + kKvBlock - 1) / kKvBlock, s.first) : 0;
    s.count = s.sink_pages + pb / kKvBlock - s.first + 1;
    return s;
}
// x / group by a product: exact for x < 2^32 / group, and a call's rows times group are under 2^28
__device__ __forceinline__ int per_group(const AttnPagedParams& p, int x) { return p.group > 1 ? (int)__umulhi((uint32_t)x, p.group_inv) : x; }
__device__ __forceinline__ bool paged_sees(const AttnPagedParams& p, int pos, int key) {
    return key <= pos && (p.window <= 0 || key > pos - p.window || key < p.sinks);
}

// Sequences of up to this many (token, head) rows per K/V head are taken page by page (paged_attn.cu), longer ones in tiles.
constexpr int kSplitRows = 32;
// Whether a call may bring a longer one
inline bool paged_prompts(const int* row_start, int rows, int max_rows, int group) {
    const long long most = max_rows > 0 && max_rows < rows ? max_rows : rows;
    return row_start && most * group > kSplitRows;
}

cudaError_t attn_paged_launch(const AttnPagedParams& p, int dtype, int row_dtype, int head_dim, int sm_count, cudaStream_t st);
size_t attn_paged_part_bytes(int sm_count);

}  // namespace mlb
