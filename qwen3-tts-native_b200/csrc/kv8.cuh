// What the kernels of the 8-bit KV cache share: the view of a cache, its codes, the span of a row's new tokens.
//
// A page of one plane (K or V) holds 16 tokens as [kv head][16][head_dim] codes, head-major like the bf16 pages, and one fp32
// scale for each head; a value is code * scale.
#pragma once

#include "q3t_common.cuh"
#include "q3t_ops.h"

#include <cuda_fp16.h>

#include <atomic>

namespace q3t {

constexpr float kKv8SmallestScale = 1.17549435e-38f;      // 2^-126: its reciprocal is finite, and neither is subnormal

struct Kv8View {
    uint8_t* k;
    uint8_t* v;
    float* k_scales;
    float* v_scales;
    long long page_stride;       // bytes
    long long scale_stride;      // elements
    int pages;
    int heads;
};

// false: the descriptor is refused
inline bool kv8_view(const Q3tKv8Cache* c, Kv8View* view) {
    if (c == nullptr || c->struct_size != sizeof(Q3tKv8Cache) || (c->format != Q3T_KV8_INT8 && c->format != Q3T_KV8_E4M3)
        || c->key_pages == nullptr || c->value_pages == nullptr || c->key_scales == nullptr || c->value_scales == nullptr
        || c->pages < 1 || c->key_value_heads < 1 || c->key_value_heads > 64 || (c->head_dimension != 64 && c->head_dimension != 128)
        || c->reserved != 0) {
        return false;
    }
    const long long page_bytes = (long long)c->key_value_heads * kPageTokens * c->head_dimension;
    view->k = c->key_pages;
    view->v = c->value_pages;
    view->k_scales = c->key_scales;
    view->v_scales = c->value_scales;
    view->page_stride = c->page_stride != 0 ? c->page_stride : page_bytes;
    view->scale_stride = c->scale_stride != 0 ? c->scale_stride : c->key_value_heads;
    view->pages = c->pages;
    view->heads = c->key_value_heads;
    const uintptr_t at = reinterpret_cast<uintptr_t>(c->key_pages) | reinterpret_cast<uintptr_t>(c->value_pages);
    const uintptr_t scales_at = reinterpret_cast<uintptr_t>(c->key_scales) | reinterpret_cast<uintptr_t>(c->value_scales);
    return view->page_stride >= page_bytes && view->page_stride % 16 == 0 && view->scale_stride >= c->key_value_heads && at % 16 == 0
           && scales_at % sizeof(float) == 0;
}

// Dynamic shared memory past what a kernel gets unasked; once a device (a bit each of `done`), and not an operation of a stream, so
// that a launch may be captured without one before it
template <class Kernel>
inline cudaError_t kv8_allow_smem(std::atomic<unsigned long long>& done, Kernel* kernel, int bytes) {
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    const unsigned long long bit = 1ull << (device & 63);
    if (e != cudaSuccess || (done.load(std::memory_order_acquire) & bit) != 0) return e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
    return e;
}

// two e4m3 codes (the low 16 bits) as fp16, exact
__device__ __forceinline__ uint32_t e4m3_to_half2(uint32_t codes) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<unsigned short>(codes)));
    return r;
}
// (lo, hi) rounded to e4m3, lo in the low byte
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// The new tokens of one row, as the device finds them, cut to what the host said of them
struct RowSpan {
    int first;        // number of its first new token
    int count;        // computed, 0 and more
    int base;         // position of the first one (negative: the row is shorter than its new tokens)
    bool cut;         // something was larger than the host said
};
__device__ __forceinline__ RowSpan row_span(const int* starts, const int* lengths, int row, int tokens, int most, int max_sequence) {
    RowSpan s;
    const int length = lengths[row];
    int from = row, to = row + 1;
    if (starts != nullptr) {
        from = starts[row];
        to = starts[row + 1];
    }
    s.first = min(max(from, 0), tokens);
    const int end = min(max(to, s.first), tokens);
    const int whole = end - s.first;
    s.count = min(whole, most);
    s.base = length - whole;
    s.cut = from != s.first || to != end || s.count != whole || length > max_sequence;
    return s;
}

// ---- attention (kv8_attention.cu, kv8_prompt.cu)

constexpr float kKv8Slack = 8.0f;         // log2 of how far a score may exceed its row's reference
constexpr float kKv8Lift = 6.0f;          // log2 of the weight at the reference
// A smaller value scale (a page of zeros has 2^-126) counts as this one where references and sums are concerned, or w / value scale would pass fp32,
// and its weights are made smaller by as much.  Values below 2^-71 so lose bits of their weights; and 2^80 is as far as others' scales
// may lie above without weights of 2^-40 of the largest leaving fp32's range.
constexpr float kKv8LeastValueScale = 8.27180613e-25f;        // 2^-80

struct Kv8AttentionArgs {
    Kv8View cache;
    const bf16* query;
    bf16* out;
    float* out32;
    const int* table;
    const int* lengths;
    const int* starts;
    int table_stride;
    int rows;
    int query_heads;
    int query_stride, out_stride;
    int tokens, most, max_sequence;
    float scale;
    void* scratch;
    int scratch_taken;        // bytes of it that are kv8_attention.cu's
    int prompts;              // a launch of kv8_prompt.cu follows
    int row_columns;          // (new tokens x query heads of a KV head) of a row up to which it is not that one's; 0: every row is, and no other launch precedes it
};

__device__ __forceinline__ float exp2_ftz(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float log2_fast(float x) {
    float r;
    asm("lg2.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float reciprocal_fast(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// 8 dims of the pieces of a column: their sum in terms of the largest reference
struct Merged {
    float top = -INFINITY, total = 0.0f, sum[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    // stats: reference and total of a piece
    __device__ __forceinline__ void add(const float2& stats, const float4& lo, const float4& hi) {
        const float most = fmaxf(top, stats.x);
        const float keep = top == -INFINITY ? 0.0f : exp2_ftz(top - most), f = stats.x == -INFINITY ? 0.0f : exp2_ftz(stats.x - most);
        const float more[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        top = most;
        total = fmaf(f, stats.y, total * keep);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] = fmaf(f, more[e], sum[e] * keep);
    }
};

// 2^n, -126 <= n <= 127
__device__ __forceinline__ float power_of_two(int n) { return __uint_as_float((uint32_t)(n + 127) << 23); }
// A query's way to fp16: times 2^shift its largest value, of which `most` is the bf16 without its sign, lies in 2^7..2^8 (or as near
// as fp32 can scale it; what is not finite stays so).  The score's scale takes it back.
__device__ __forceinline__ int query_shift(uint32_t most) { return min(134 - (int)min(most >> 7, 254u), 127); }
__device__ __forceinline__ float query_back(float scale, int shift) {
    const int half = shift / 2;
    return scale * power_of_two(-half) * power_of_two(half - shift);
}
// four codes as two pairs of fp16
template <bool E4M3>
__device__ __forceinline__ void codes_to_half(uint32_t word, uint32_t& lo, uint32_t& hi) {
    if (E4M3) {
        lo = e4m3_to_half2(word);
        hi = e4m3_to_half2(word >> 16);
    } else {
        // the byte behind 0x64 is 1024 + it as fp16, with its sign bit turned over 1152 + the code
        const uint32_t biased = word ^ 0x80808080u;
        const __half2 offset = __half2half2(__ushort_as_half(0x6480));
        const uint32_t a = __byte_perm(biased, 0x64646464u, 0x4140), b = __byte_perm(biased, 0x64646464u, 0x4342);
        const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), offset), y = __hsub2(*reinterpret_cast<const __half2*>(&b), offset);
        lo = *reinterpret_cast<const uint32_t*>(&x);
        hi = *reinterpret_cast<const uint32_t*>(&y);
    }
}

}  // namespace q3t
