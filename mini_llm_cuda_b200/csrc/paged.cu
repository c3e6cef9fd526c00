// Operators over a caller's paged K/V cache: the handle, the rotating append, the read, and the entry point of the attention (its
// kernels are in paged_attn.cu).
#include <algorithm>
#include <cmath>
#include <new>

#include "errors.h"
#include "paged.cuh"

using namespace mlb;

struct mlb_ops {
    int device = 0, sm_count = 0;
    unsigned char* mem = nullptr;       // error word | plan of the split attention | its partial results
};

namespace {

constexpr size_t kOpsErrBytes = 256;
constexpr int kOpsMaxBatch = 4096, kOpsMaxHeads = 65535;      // (of K/V: a dimension of a grid)
constexpr size_t kOpsPlanBytes = ((kOpsMaxBatch + 1) * 8 + 255) / 256 * 256;

// The handle's device is current while an object of this lives.
struct OnDevice {
    int before = -1, now = -1;
    cudaError_t err;
    explicit OnDevice(int device) : now(device) {
        err = cudaGetDevice(&before);
        if (err == cudaSuccess && before != device) err = cudaSetDevice(device);
    }
    ~OnDevice() {
        if (before >= 0 && before != now) cudaSetDevice(before);
    }
};

#define CU(expr)                                                                              \
    do {                                                                                      \
        cudaError_t e__ = (expr);                                                             \
        if (e__ != cudaSuccess)                                                               \
            return fail(MLB_E_CUDA, "%s failed: %s (%s:%d)", #expr, cudaGetErrorString(e__), __FILE__, __LINE__); \
    } while (0)

int check_cache(const char* op, const mlb_paged_kv* kv, const mlb_new_rows* r, int row_dtype) {
    if (!kv || !r) return fail(MLB_E_INVALID, "%s: null pointer", op);
    if (!kv->kpool || !kv->vpool || !kv->page_table || !r->kv_lens) return fail(MLB_E_INVALID, "%s: null pointer in the cache or the rows", op);
    if (kv->dtype != MLB_DT_F32 && kv->dtype != MLB_DT_BF16 && kv->dtype != MLB_DT_FP4_E2M1)
        return fail(MLB_E_INVALID, "%s: a cache is float32, bfloat16 or fp4_e2m1", op);
    if (row_dtype != MLB_DT_F32 && row_dtype != MLB_DT_BF16) return fail(MLB_E_INVALID, "%s: rows are float32 or bfloat16", op);
    if (kv->dtype == MLB_DT_FP4_E2M1) {
        if (!kv->kscale || !kv->vscale) return fail(MLB_E_INVALID, "%s: a 4-bit cache has scales", op);
        if (!(kv->k_scale > 0.f) || !(kv->v_scale > 0.f) || !std::isfinite(kv->k_scale) || !std::isfinite(kv->v_scale))
            return fail(MLB_E_INVALID, "%s: k_scale and v_scale are positive numbers", op);
    }
    if (kv->pt_stride < 1 || kv->num_pages < 1 || kv->kv_heads < 1) return fail(MLB_E_INVALID, "%s: pt_stride, num_pages and kv_heads must be >= 1", op);
    if (kv->pt_stride > (1 << 26)) return fail(MLB_E_UNSUPPORTED, "%s: pt_stride above 2^26 (positions are 31-bit numbers)", op);
    if (kv->kv_heads > kOpsMaxHeads) return fail(MLB_E_UNSUPPORTED, "%s: kv_heads above %d", op, kOpsMaxHeads);
    if (kv->head_dim != 64 && kv->head_dim != 128) return fail(MLB_E_UNSUPPORTED, "%s: head_dim must be 64 or 128", op);
    if ((reinterpret_cast<uintptr_t>(kv->kpool) | reinterpret_cast<uintptr_t>(kv->vpool)) & 15) return fail(MLB_E_INVALID, "%s: pools start on 16 bytes", op);
    if (kv->dtype == MLB_DT_FP4_E2M1 && ((reinterpret_cast<uintptr_t>(kv->kscale) | reinterpret_cast<uintptr_t>(kv->vscale)) & 15))
        return fail(MLB_E_INVALID, "%s: scales start on 16 bytes", op);
    if (r->batch < 1 || r->batch > kOpsMaxBatch) return fail(MLB_E_INVALID, "%s: batch must be in 1..%d", op, kOpsMaxBatch);
    if (r->rows < 0 || r->max_rows < 0) return fail(MLB_E_INVALID, "%s: rows and max_rows must be >= 0", op);
    return MLB_OK;
}

// Rows of `width` elements each: present, on their type's boundary, not overlapping
int check_rows(const char* op, const char* what, const void* p, int64_t stride, int64_t width, int row_dtype, int rows) {
    if (rows == 0) return MLB_OK;
    if (!p) return fail(MLB_E_INVALID, "%s: null %s", op, what);
    if (reinterpret_cast<uintptr_t>(p) % (row_dtype == MLB_DT_F32 ? 4 : 2)) return fail(MLB_E_INVALID, "%s: %s is not on its type's boundary", op, what);
    if (stride < width && rows > 1) return fail(MLB_E_INVALID, "%s: the stride of %s is smaller than its row", op, what);
    return MLB_OK;
}

// The handle, and sizes that the kernels' 31-bit row and thread numbers hold
int check_count(const char* op, const mlb_ops* o, const mlb_new_rows* r, long long heads, int head_dim) {
    if (r->rows * heads * (head_dim / 8) > (1LL << 30)) return fail(MLB_E_UNSUPPORTED, "%s: too many rows for one call", op);
    if (!o) return fail(MLB_E_INVALID, "%s: null handle", op);
    return MLB_OK;
}

PagedCache cache_of(const mlb_paged_kv* kv) {
    PagedCache c;
    c.kpool = kv->kpool; c.vpool = kv->vpool;
    c.kscale = static_cast<unsigned char*>(kv->kscale); c.vscale = static_cast<unsigned char*>(kv->vscale);
    c.page_table = kv->page_table; c.pt_stride = kv->pt_stride; c.num_pages = kv->num_pages; c.kv_heads = kv->kv_heads;
    c.k_scale = kv->dtype == MLB_DT_FP4_E2M1 ? kv->k_scale : 1.f;
    c.v_scale = kv->dtype == MLB_DT_FP4_E2M1 ? kv->v_scale : 1.f;
    return c;
}
PagedRows rows_of(const mlb_ops* o, const mlb_new_rows* r) {
    PagedRows p;
    p.row_start = r->row_start; p.kv_lens = r->kv_lens; p.batch = r->batch; p.rows = r->rows; p.max_rows = r->max_rows;
    p.err = reinterpret_cast<int*>(o->mem);
    return p;
}

// ---- append and read ---------------------------------------------------------------------------------------------
// A CTA takes up to kMoveRows rows. Its warps look up where these stand (sequence, position, page) first, a row each. Then a thread takes eight dims
// (16 bytes of bf16 rows, 32 of fp32) of one head of all of the rows, so that what depends on the head alone is worked out once, and goes on to
// another head where there are more than the CTA's threads hold. K heads first, then V heads, then (append) the query heads. Bound by HBM, or by the
// launch. A thread per eight dims of the call, each of which looked up its own row, executed 300 instructions for them and was bound by
// these: 125 us for 16001 rows of 32 + 2 x 8 heads of 128, bf16, into 4 bits, and 37 us to read K and V back; 76 and 23 this way, 4.7 and 3.7 TB/s.
constexpr int kMoveThreads = 256, kMoveRows = 8;

struct MoveParams {
    PagedCache c;
    PagedRows r;
    const void *k, *v, *q;
    void *k_out, *v_out, *q_out;
    long long k_stride, v_stride, q_stride;      // of whichever of in / out is the caller's
    long long q_out_stride;
    const float* rope; int rope_len;
    int heads;                                   // query heads, 0 without them
    int vec;                                     // all rows (and the table) start on 16 bytes
    int cta_rows;                                // rows of a CTA
};

// Eight numbers as they lie in memory
template <typename RT>
struct Raw8 {
    uint4 w[sizeof(RT) / 2];
    __device__ __forceinline__ void load(const RT* p, bool vec) {
        if (vec) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(RT) / 2; ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
        } else if constexpr (sizeof(RT) == 2) {
            uint32_t u[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] = (uint32_t)__bfloat16_as_ushort(p[2 * i]) | (uint32_t)__bfloat16_as_ushort(p[2 * i + 1]) << 16;
            w[0] = make_uint4(u[0], u[1], u[2], u[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                w[i] = make_uint4(__float_as_uint(p[4 * i]), __float_as_uint(p[4 * i + 1]), __float_as_uint(p[4 * i + 2]), __float_as_uint(p[4 * i + 3]));
        }
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
        if constexpr (sizeof(RT) == 2) {
            const uint32_t u[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[2 * i] = __uint_as_float(u[i] << 16);
                x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                x[4 * i] = __uint_as_float(w[i].x); x[4 * i + 1] = __uint_as_float(w[i].y);
                x[4 * i + 2] = __uint_as_float(w[i].z); x[4 * i + 3] = __uint_as_float(w[i].w);
            }
        }
    }
};
template <typename RT>
__device__ __forceinline__ void store8(RT* p, bool vec, const float (&x)[8]) {
    if (vec) {
        if (sizeof(RT) == 2) {
            uint32_t u[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                u[i] = f32x2_to_bf16(x[2 * i], x[2 * i + 1]);
            }
            *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
        } else {
            reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
            reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) Elem<RT>::put(p, i, x[i]);
    }
}

// Sequence of row t: the last b with row_start[b] <= t (empty sequences before it have the same start), 32 probes a round by one warp
__device__ __forceinline__ int find_seq(const int* row_start, int batch, int t) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = batch;                      // answer in [lo, hi)
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, at = lo + lane * step;
        const unsigned le = __ballot_sync(0xffffffffu, at < hi && row_start[at] <= t);
        const int n = __popc(le);                // (of a sequence that does not increase: some number)
        if (n == 0) return lo;
        lo += (n - 1) * step;
        hi = min(hi, lo + step);
    }
    return lo;
}

template <typename KVT, typename RT, int HD, bool READ>
__global__ void __launch_bounds__(kMoveThreads, 4) kv_move_kernel(const __grid_constant__ MoveParams p) {
    constexpr int PER = HD / 8;                  // threads of a head
    constexpr bool Q4 = sizeof(KVT) == 1;
    __shared__ int place[kMoveRows];             // position; negative: nothing to do
    __shared__ long long pool_row[kMoveRows];    // row of the pools, of head 0; negative: none to write to
    __shared__ float4 turns[READ ? 1 : kMoveRows][2][PER];        // the rows' (cos, sin): first four and last four of a thread's eight numbers
    const int tid = threadIdx.x, first = (int)blockIdx.x * p.cta_rows, n = min(p.cta_rows, p.r.rows - first);
    for (int i = tid / 32; i < n; i += (int)blockDim.x / 32) {
        const int t = first + i, b = p.r.row_start ? find_seq(p.r.row_start, p.r.batch, t) : t;
        if (tid % 32 == 0) {
            int pos = -1, page = -1;
            if (b < p.r.batch) {
                const PagedSeq s = paged_seq(p.r, p.c.pt_stride, b, true);
                if (t >= s.r0 && t < s.r0 + s.n) pos = s.len - s.n + (t - s.r0);
            }
            if (!READ && p.rope && pos >= p.rope_len) {
                atomicExch(p.r.err, PG_ROPE);
                pos = -1;
            }
            if (pos >= 0) page = paged_page(p.c, p.r.err, b, pos / kKvBlock, READ ? 0 : -1);
            place[i] = pos;
            pool_row[i] = page < 0 ? -1 : (long long)page * p.c.kv_heads * kKvBlock + pos % kKvBlock;
        }
    }
    __syncthreads();
    const bool vec = p.vec != 0;
    if (!READ && p.rope) {
        for (int i = tid; i < n * PER; i += (int)blockDim.x) {
            const int r = i / PER, c = i % PER;
            if (place[r] < 0) continue;
            Raw8<float> w;
            float x[8];
            w.load(p.rope + (size_t)place[r] * HD + c * 8, vec);
            w.get(x);
            turns[r][0][c] = make_float4(x[0], x[1], x[2], x[3]);
            turns[r][1][c] = make_float4(x[4], x[5], x[6], x[7]);
        }
        __syncthreads();
    }
    const int heads = 2 * p.c.kv_heads + (READ ? 0 : p.heads), e = tid % PER * 8;
    for (int h0 = 0; h0 < heads; h0 += (int)blockDim.x / PER) {
        const int head = h0 + tid / PER;
        const bool in = head < heads, is_k = head < p.c.kv_heads, is_v = !is_k && head < 2 * p.c.kv_heads, pooled = is_k || is_v;
        const int h = is_k ? head : is_v ? head - p.c.kv_heads : head - 2 * p.c.kv_heads;
        // this thread's place in row `first` of the caller's tensor, and in row 0 of the head's in a page
        const long long stride = is_k ? p.k_stride : is_v ? p.v_stride : p.q_stride;
        const size_t at = first * stride + h * HD + e;
        unsigned char* const pool = static_cast<unsigned char*>(is_k ? p.c.kpool : p.c.vpool) + (Q4 ? ((size_t)h * kKvBlock * HD + e) / 2 : ((size_t)h * kKvBlock * HD + e) * sizeof(KVT));
        unsigned char* const scales = Q4 ? (is_k ? p.c.kscale : p.c.vscale) + ((size_t)h * kKvBlock * HD + e) / 16 : nullptr;
        const float g = is_k ? p.c.k_scale : p.c.v_scale;
        if constexpr (READ) {
            RT* dst = static_cast<RT*>(is_k ? p.k_out : p.v_out) + at;
            if (!in) break;
#pragma unroll 4
            for (int i = 0; i < n; ++i, dst += stride) {
                if (place[i] < 0) continue;
                const size_t row = (size_t)pool_row[i];
                float x[8];
                if constexpr (Q4) {
                    const uint32_t codes = __ldg(reinterpret_cast<const uint32_t*>(pool + row * (HD / 2)));
                    const float s = e4m3_to_f32(__ldg(scales + row * (HD / 16)));
                    uint32_t w[4];
                    e2m1x8_to_f16(codes, w);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        x[2 * j] = __fmul_rn(__fmul_rn(f16_lo(w[j]), s), g);
                        x[2 * j + 1] = __fmul_rn(__fmul_rn(f16_hi(w[j]), s), g);
                    }
                } else {
                    Raw8<KVT> raw;
                    raw.load(reinterpret_cast<const KVT*>(pool) + row * HD, true);
                    raw.get(x);
                }
                store8(dst, vec, x);
            }
        } else {
            const bool turn = p.rope && !is_v;
            const bool some_pooled = __any_sync(0xffffffffu, in && pooled);
            const RT* src = static_cast<const RT*>(is_k ? p.k : is_v ? p.v : p.q) + at;
            RT* dst = static_cast<RT*>(p.q_out) + (first * p.q_out_stride + h * HD + e);
            auto put = [&](int i, float (&x)[8]) {
                if (i >= n || place[i] < 0) return;              // (the whole CTA: 4-bit pages take shuffles)
                if (turn) {
                    const float4 c0 = turns[i][0][tid % PER], c1 = turns[i][1][tid % PER];
                    const float cs[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        const float a = x[j], c = x[j + 1];
                        x[j] = __fsub_rn(__fmul_rn(cs[j], a), __fmul_rn(cs[j + 1], c));
                        x[j + 1] = __fadd_rn(__fmul_rn(cs[j + 1], a), __fmul_rn(cs[j], c));
                    }
                }
                const long long row = pool_row[i];
                if constexpr (Q4) {
                    if (some_pooled) {
                        // two neighbouring threads hold the 16 values of a scale
                        float top = 0.f;
#pragma unroll
                        for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(x[j]));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                        if (in && pooled && row >= 0) {
                            const unsigned char s = f32_to_e4m3(__fdiv_rn(top, __fmul_rn(6.f, g)));
                            const float unit = __fmul_rn(e4m3_to_f32(s), g), inv = unit > 0.f ? __fdiv_rn(1.f, unit) : 0.f;
                            float y[8];
#pragma unroll
                            for (int j = 0; j < 8; ++j) y[j] = __fmul_rn(x[j], inv);
                            *reinterpret_cast<uint32_t*>(pool + row * (HD / 2)) = f32x8_to_e2m1(y);
                            if (e % 16 == 0) scales[row * (HD / 16)] = s;
                        }
                    }
                } else if (in && pooled && row >= 0) {
                    store8(reinterpret_cast<KVT*>(pool) + row * HD, true, x);
                }
                if (in && !pooled) store8(dst + i * p.q_out_stride, vec, x);
            };
            // several rows at a time, so that the loads of all are on their way
            constexpr int U = 4;
            for (int i = 0; i < n; i += U) {
                Raw8<RT> raw[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (i + u >= n || place[i + u] < 0 || !in) continue;
                    raw[u].load(src + (i + u) * stride, vec);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    float x[8];
                    raw[u].get(x);
                    put(i + u, x);
                }
            }
        }
    }
}

template <bool READ, typename KVT, typename RT>
cudaError_t move_launch(MoveParams p, int hd, int sm_count, cudaStream_t st) {
    // threads for the heads of a row, or a part of them; more rows of a CTA where there are enough for eight CTAs on each SM
    const int units = (2 * p.c.kv_heads + (READ ? 0 : p.heads)) * (hd / 8);
    const int threads = std::min(kMoveThreads, (units + 31) / 32 * 32);
    p.cta_rows = std::max(1, std::min(kMoveRows, p.r.rows / (8 * sm_count)));
    const unsigned ctas = (unsigned)((p.r.rows + p.cta_rows - 1) / p.cta_rows);
    if (hd == 64) kv_move_kernel<KVT, RT, 64, READ><<<ctas, threads, 0, st>>>(p);
    else kv_move_kernel<KVT, RT, 128, READ><<<ctas, threads, 0, st>>>(p);
    return cudaGetLastError();
}
template <bool READ>
cudaError_t move_types(const MoveParams& p, int dtype, int row_dtype, int hd, int sm_count, cudaStream_t st) {
    const bool f = row_dtype == MLB_DT_F32;
    if (dtype == MLB_DT_F32) return f ? move_launch<READ, float, float>(p, hd, sm_count, st) : move_launch<READ, float, bf16_t>(p, hd, sm_count, st);
    if (dtype == MLB_DT_BF16) return f ? move_launch<READ, bf16_t, float>(p, hd, sm_count, st) : move_launch<READ, bf16_t, bf16_t>(p, hd, sm_count, st);
    return f ? move_launch<READ, fp4_t, float>(p, hd, sm_count, st) : move_launch<READ, fp4_t, bf16_t>(p, hd, sm_count, st);
}

bool on16(const void* p, int64_t stride, int elt) { return ((reinterpret_cast<uintptr_t>(p) | (uint64_t)stride * elt) & 15) == 0; }

}  // namespace

extern "C" int mlb_ops_new(int device, mlb_ops** out) {
    if (!out) return fail(MLB_E_INVALID, "null argument");
    *out = nullptr;
    int n = 0;
    CU(cudaGetDeviceCount(&n));
    if (device < 0 || device >= n) return fail(MLB_E_INVALID, "device %d: there are %d", device, n);
    OnDevice on(device);
    CU(on.err);
    mlb_ops* o = new (std::nothrow) mlb_ops;
    if (!o) return fail(MLB_E_NOMEM, "out of host memory");
    o->device = device;
    cudaError_t e = cudaDeviceGetAttribute(&o->sm_count, cudaDevAttrMultiProcessorCount, device);
    if (e == cudaSuccess) e = cudaMalloc(reinterpret_cast<void**>(&o->mem), kOpsErrBytes + kOpsPlanBytes + attn_paged_part_bytes(o->sm_count));
    if (e == cudaSuccess) e = cudaMemset(o->mem, 0, kOpsErrBytes);
    if (e == cudaSuccess) e = cudaDeviceSynchronize();         // the caller's streams do not wait for the default stream
    if (e != cudaSuccess) {
        cudaFree(o->mem);
        delete o;
        return fail(e == cudaErrorMemoryAllocation ? MLB_E_NOMEM : MLB_E_CUDA, "mlb_ops_new: %s", cudaGetErrorString(e));
    }
    *out = o;
    return MLB_OK;
}

extern "C" void mlb_ops_free(mlb_ops* o) {
    if (!o) return;
    OnDevice on(o->device);
    cudaFree(o->mem);
    delete o;
}

extern "C" int mlb_ops_status(mlb_ops* o, void* stream) {
    if (!o) return fail(MLB_E_INVALID, "null argument");
    OnDevice on(o->device);
    CU(on.err);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int code = 0;
    CU(cudaMemcpyAsync(&code, o->mem, 4, cudaMemcpyDeviceToHost, st));
    CU(cudaStreamSynchronize(st));
    if (code == 0) return MLB_OK;
    CU(cudaMemsetAsync(o->mem, 0, 4, st));
    CU(cudaStreamSynchronize(st));
    switch (code) {
        case PG_ROWS: return fail(MLB_E_INVALID, "paged operator: row_start is no increasing sequence in 0..rows");
        case PG_MAX_ROWS: return fail(MLB_E_INVALID, "paged operator: a sequence brings more rows than max_rows");
        case PG_LONG: return fail(MLB_E_INVALID, "paged operator: a sequence needs more pages than pt_stride");
        case PG_PAGE: return fail(MLB_E_INVALID, "paged operator: the page table names a page outside [0, num_pages)");
        case PG_ROPE: return fail(MLB_E_INVALID, "paged operator: a position lies behind the rotation table");
        default: return fail(MLB_E_TIMEOUT, "paged operator: a bounded wait ran out (code %d)", code);
    }
}

extern "C" int mlb_op_kv_append(mlb_ops* o, const mlb_paged_kv* kv, const mlb_new_rows* rows, int row_dtype, const void* k, int64_t k_stride,
                                const void* v, int64_t v_stride, const float* rope_or_null, int rope_len, const void* q_or_null,
                                int64_t q_stride, void* q_out, int64_t q_out_stride, int heads, void* stream) {
    int rc = check_cache("append", kv, rows, row_dtype);
    if (rc) return rc;
    const int64_t width = (int64_t)kv->kv_heads * kv->head_dim;
    if ((rc = check_rows("append", "k", k, k_stride, width, row_dtype, rows->rows))) return rc;
    if ((rc = check_rows("append", "v", v, v_stride, width, row_dtype, rows->rows))) return rc;
    if (rope_or_null && (rope_len < 1 || reinterpret_cast<uintptr_t>(rope_or_null) % 4)) return fail(MLB_E_INVALID, "append: a rotation table has rows of fp32");
    if (q_or_null) {
        if (heads < 1) return fail(MLB_E_INVALID, "append: heads must be >= 1");
        if (heads > 8 * kOpsMaxHeads) return fail(MLB_E_UNSUPPORTED, "append: heads above %d", 8 * kOpsMaxHeads);
        if ((rc = check_rows("append", "q", q_or_null, q_stride, (int64_t)heads * kv->head_dim, row_dtype, rows->rows))) return rc;
        if ((rc = check_rows("append", "q_out", q_out, q_out_stride, (int64_t)heads * kv->head_dim, row_dtype, rows->rows))) return rc;
    }
    if (q_or_null && q_or_null == q_out && q_stride != q_out_stride && rows->rows > 1)
        return fail(MLB_E_INVALID, "append: q_out may be q with the same stride, and not overlap it otherwise");
    if ((rc = check_count("append", o, rows, 2LL * kv->kv_heads + (q_or_null ? heads : 0), kv->head_dim))) return rc;
    if (rows->rows == 0) return MLB_OK;
    const int elt = row_dtype == MLB_DT_F32 ? 4 : 2;
    MoveParams p{};
    p.c = cache_of(kv);
    p.r = rows_of(o, rows);
    p.k = k; p.k_stride = k_stride; p.v = v; p.v_stride = v_stride;
    p.rope = rope_or_null; p.rope_len = rope_len;
    p.vec = on16(k, k_stride, elt) && on16(v, v_stride, elt) && on16(rope_or_null, 0, 4);
    if (q_or_null) {
        p.q = q_or_null; p.q_stride = q_stride; p.q_out = q_out; p.q_out_stride = q_out_stride; p.heads = heads;
        p.vec = p.vec && on16(q_or_null, q_stride, elt) && on16(q_out, q_out_stride, elt);
    }
    OnDevice on(o->device);
    CU(on.err);
    CU(move_types<false>(p, kv->dtype, row_dtype, kv->head_dim, o->sm_count, static_cast<cudaStream_t>(stream)));
    return MLB_OK;
}

extern "C" int mlb_op_kv_read(mlb_ops* o, const mlb_paged_kv* kv, const mlb_new_rows* rows, int row_dtype, void* k_out, int64_t k_stride,
                              void* v_out, int64_t v_stride, void* stream) {
    int rc = check_cache("read", kv, rows, row_dtype);
    if (rc) return rc;
    const int64_t width = (int64_t)kv->kv_heads * kv->head_dim;
    if ((rc = check_rows("read", "k_out", k_out, k_stride, width, row_dtype, rows->rows))) return rc;
    if ((rc = check_rows("read", "v_out", v_out, v_stride, width, row_dtype, rows->rows))) return rc;
    if ((rc = check_count("read", o, rows, 2LL * kv->kv_heads, kv->head_dim))) return rc;
    if (rows->rows == 0) return MLB_OK;
    const int elt = row_dtype == MLB_DT_F32 ? 4 : 2;
    MoveParams p{};
    p.c = cache_of(kv);
    p.r = rows_of(o, rows);
    p.k_out = k_out; p.k_stride = k_stride; p.v_out = v_out; p.v_stride = v_stride;
    p.vec = on16(k_out, k_stride, elt) && on16(v_out, v_stride, elt);
    OnDevice on(o->device);
    CU(on.err);
    CU(move_types<true>(p, kv->dtype, row_dtype, kv->head_dim, o->sm_count, static_cast<cudaStream_t>(stream)));
    return MLB_OK;
}

extern "C" int mlb_op_attn_paged(mlb_ops* o, const mlb_paged_kv* kv, const mlb_new_rows* rows, int row_dtype, const void* q, int64_t q_stride,
                                 const float* gate_or_null, void* out, int64_t out_stride, int heads, float scale, int window, int sinks,
                                 void* stream) {
    int rc = check_cache("paged attention", kv, rows, row_dtype);
    if (rc) return rc;
    if (heads < 1 || heads % kv->kv_heads) return fail(MLB_E_INVALID, "paged attention: heads must be a multiple of kv_heads");
    if (heads / kv->kv_heads > 8) return fail(MLB_E_UNSUPPORTED, "paged attention: at most 8 query heads per K/V head");
    if (window < 0 || sinks < 0) return fail(MLB_E_INVALID, "paged attention: window and sinks must be >= 0");
    if (!std::isfinite(scale)) return fail(MLB_E_INVALID, "paged attention: scale must be a number");
    if ((rc = check_rows("paged attention", "q", q, q_stride, (int64_t)heads * kv->head_dim, row_dtype, rows->rows))) return rc;
    if ((rc = check_rows("paged attention", "out", out, out_stride, (int64_t)heads * kv->head_dim, row_dtype, rows->rows))) return rc;
    if (gate_or_null && reinterpret_cast<uintptr_t>(gate_or_null) % 4) return fail(MLB_E_INVALID, "paged attention: gate is not on its type's boundary");
    // prompts: a row of a bf16 pool is a coordinate of a tensor map, a 31-bit number
    if (kv->dtype == MLB_DT_BF16 && row_dtype == MLB_DT_BF16 && paged_prompts(rows->row_start, rows->rows, rows->max_rows, heads / kv->kv_heads) &&
        (long long)kv->num_pages * kv->kv_heads > 0x7fffffffLL / kKvBlock)
        return fail(MLB_E_UNSUPPORTED, "paged attention: prompts over bfloat16 pages take pools of less than 2^31 rows of a head");
    if ((rc = check_count("paged attention", o, rows, heads, kv->head_dim))) return rc;
    if (rows->rows > 0 && q == out) return fail(MLB_E_INVALID, "paged attention: out may not be q");
    if (rows->rows == 0) return MLB_OK;
    AttnPagedParams p{};
    p.c = cache_of(kv);
    p.r = rows_of(o, rows);
    p.q = q; p.q_stride = q_stride; p.gate = gate_or_null; p.out = out; p.out_stride = out_stride;
    p.heads = heads; p.group = heads / kv->kv_heads;
    p.group_inv = p.group > 1 ? (uint32_t)((1ull << 32) / (uint32_t)p.group + 1) : 0;
    p.scale = scale != 0.f ? scale : 1.f / std::sqrt((float)kv->head_dim);
    p.window = std::min(window, 1 << 30);        // no position reaches that far (pt_stride), and differences stay within 32 bits
    p.sinks = std::min(sinks, 1 << 30);
    p.plan = reinterpret_cast<unsigned long long*>(o->mem + kOpsErrBytes);
    p.part = reinterpret_cast<float*>(o->mem + kOpsErrBytes + kOpsPlanBytes);
    OnDevice on(o->device);
    CU(on.err);
    CU(attn_paged_launch(p, kv->dtype, row_dtype, kv->head_dim, o->sm_count, static_cast<cudaStream_t>(stream)));
    return MLB_OK;
}
