// Causal attention over an 8-bit paged cache (q3t_launch_kv8_attention).
//
// out = sum_j w_j v_j / sum_j w_j, w_j = exp(scale * q . k_j - max), over the positions up to the token's own.  One CTA a token and
// query head, its warps taking pages in turn: the plain kernel, right for every shape.

#include "kv8.cuh"
#include "q3t_kernels.cuh"

#include <climits>

namespace q3t {
namespace {

constexpr int kSimpleThreads = 128;
constexpr int kSimpleWarps = kSimpleThreads / kWarp;

__device__ unsigned int g_kv8_range_errors = 0;
__device__ unsigned int g_kv8_page_errors = 0;

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
};

template <int HD, bool E4M3>
__global__ void __launch_bounds__(kSimpleThreads) kv8_attention_simple_kernel(const Kv8AttentionArgs a) {
    constexpr int kPer = HD / kWarp;          // dims a lane
    __shared__ float part[kSimpleWarps][HD + 2];
    const int lane = threadIdx.x % kWarp, warp = threadIdx.x / kWarp;
    const int row = blockIdx.y, head = blockIdx.z;
    const RowSpan span = row_span(a.starts, a.lengths, row, a.tokens, a.most, a.max_sequence);
    if (span.cut && blockIdx.x == 0 && head == 0 && threadIdx.x == 0) atomicAdd(&g_kv8_range_errors, 1u);
    const int kv_head = head / (a.query_heads / a.cache.heads);
    for (int i = blockIdx.x; i < span.count; i += gridDim.x) {
        const int token = span.first + i;
        const int seen = min(max(span.base + i + 1, 0), a.max_sequence);
        float q[kPer], o[kPer], top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int d = 0; d < kPer; ++d) {
            q[d] = bf2f(a.query[(size_t)token * a.query_stride + (size_t)head * HD + lane * kPer + d]) * a.scale;
            o[d] = 0.0f;
        }
        for (int page = warp; page * kPageTokens < seen; page += kSimpleWarps) {
            const int id = a.table[(size_t)row * a.table_stride + page];
            if (id < 0 || id >= a.cache.pages) {
                if (lane == 0 && head == 0 && i == 0) atomicAdd(&g_kv8_page_errors, 1u);
                continue;
            }
            const size_t at = (size_t)id * a.cache.page_stride + (size_t)kv_head * (kPageTokens * HD) + lane * kPer;
            const float ks = a.cache.k_scales[(size_t)id * a.cache.scale_stride + kv_head];
            const float vs = a.cache.v_scales[(size_t)id * a.cache.scale_stride + kv_head];
            auto value = [&](const uint8_t* plane, int t, int d) {
                const uint8_t c = plane[at + t * HD + d];
                if (!E4M3) return static_cast<float>(static_cast<signed char>(c));
                const uint32_t h = e4m3_to_half2(c);
                return __low2float(*reinterpret_cast<const __half2*>(&h));
            };
            for (int t = 0; t < min(kPageTokens, seen - page * kPageTokens); ++t) {
                float s = 0.0f;
#pragma unroll
                for (int d = 0; d < kPer; ++d) s = fmaf(q[d], value(a.cache.k, t, d), s);
                s = warp_sum_xor(s) * ks;
                const float now = fmaxf(top, s);
                const float keep = now == -INFINITY ? 1.0f : expf(top - now), w = now == -INFINITY ? 0.0f : expf(s - now);
                top = now;
                sum = sum * keep + w;
#pragma unroll
                for (int d = 0; d < kPer; ++d) o[d] = o[d] * keep + w * vs * value(a.cache.v, t, d);
            }
        }
        __syncthreads();
#pragma unroll
        for (int d = 0; d < kPer; ++d) part[warp][lane * kPer + d] = o[d];
        if (lane == 0) {
            part[warp][HD] = top;
            part[warp][HD + 1] = sum;
        }
        __syncthreads();
        if (threadIdx.x < HD) {
            float all = -INFINITY, total = 0.0f, out = 0.0f;
            for (int w = 0; w < kSimpleWarps; ++w) all = fmaxf(all, part[w][HD]);
            for (int w = 0; w < kSimpleWarps; ++w) {
                const float f = part[w][HD] == -INFINITY ? 0.0f : expf(part[w][HD] - all);
                total += f * part[w][HD + 1];
                out += f * part[w][threadIdx.x];
            }
            out = total > 0.0f || total != total ? out / total : 0.0f;
            a.out[(size_t)token * a.out_stride + (size_t)head * HD + threadIdx.x] = f2bf(out);
            if (a.out32 != nullptr) a.out32[((size_t)token * a.query_heads + head) * HD + threadIdx.x] = out;
        }
    }
}

// false: refused
bool attention_args(const Q3tKv8AttentionDesc* d, Kv8AttentionArgs* a) {
    if (d == nullptr || d->struct_size != sizeof(Q3tKv8AttentionDesc) || !kv8_view(d->cache, &a->cache)) return false;
    const Q3tKv8Cache& c = *d->cache;
    if (d->rows < 1 || d->rows > Q3T_MAX_TABLE_ROWS || d->query == nullptr || d->output == nullptr || d->page_table == nullptr
        || d->lengths == nullptr || d->page_table_stride < 1 || d->query_heads < 1 || d->query_heads % c.key_value_heads != 0
        || d->query_heads / c.key_value_heads > 64 || d->tokens < 0 || d->max_row_tokens < 0 || d->max_sequence_length < 1
        || (d->max_sequence_length - 1) / kPageTokens >= d->page_table_stride || !(d->scale >= 0.0f)) {
        return false;
    }
    // one token a row
    if (d->token_starts == nullptr && (d->tokens < d->rows || d->max_row_tokens < 1)) return false;
    const int width = d->query_heads * c.head_dimension;
    a->query_stride = d->query_stride != 0 ? d->query_stride : width;
    a->out_stride = d->output_stride != 0 ? d->output_stride : width;
    if (a->query_stride < width || a->out_stride < width || a->query_stride % 8 != 0 || a->out_stride % 8 != 0
        || (reinterpret_cast<uintptr_t>(d->query) | reinterpret_cast<uintptr_t>(d->output) | reinterpret_cast<uintptr_t>(d->output_f32)) % 16 != 0) {
        return false;
    }
    a->query = reinterpret_cast<const bf16*>(d->query);
    a->out = reinterpret_cast<bf16*>(d->output);
    a->out32 = d->output_f32;
    a->table = d->page_table;
    a->lengths = d->lengths;
    a->starts = d->token_starts;
    a->table_stride = d->page_table_stride;
    a->rows = d->rows;
    a->query_heads = d->query_heads;
    a->tokens = d->tokens;
    a->most = d->max_row_tokens < d->tokens ? d->max_row_tokens : d->tokens;
    a->max_sequence = d->max_sequence_length;
    a->scale = d->scale > 0.0f ? d->scale : 1.0f / sqrtf(static_cast<float>(c.head_dimension));
    return true;
}

}  // namespace

unsigned int kv8_append_page_error_count();
unsigned int kv8_range_error_count() {
    unsigned int v = 0;
    return cudaMemcpyFromSymbol(&v, g_kv8_range_errors, sizeof(v)) == cudaSuccess ? v : ~0u;
}

}  // namespace q3t

extern "C" uint32_t q3t_kv8_page_error_count(void) {
    unsigned int v = 0;
    return cudaMemcpyFromSymbol(&v, q3t::g_kv8_page_errors, sizeof(v)) == cudaSuccess ? v + q3t::kv8_append_page_error_count() : ~0u;
}

extern "C" size_t q3t_kv8_attention_scratch_bytes(const Q3tKv8AttentionDesc* desc) {
    q3t::Kv8AttentionArgs a;
    return q3t::attention_args(desc, &a) ? 16 : 0;
}

extern "C" int32_t q3t_launch_kv8_attention(const Q3tKv8AttentionDesc* desc, void* stream) {
    using namespace q3t;
    Kv8AttentionArgs a;
    if (!attention_args(desc, &a) || desc->scratch == nullptr || reinterpret_cast<uintptr_t>(desc->scratch) % 16 != 0
        || desc->scratch_bytes < q3t_kv8_attention_scratch_bytes(desc)) {
        return cudaErrorInvalidValue;
    }
    if (a.most == 0) return cudaSuccess;
    const dim3 grid((unsigned)min(a.most, 65536), (unsigned)a.rows, (unsigned)a.query_heads);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool e4m3 = desc->cache->format == Q3T_KV8_E4M3;
    auto* kernel = desc->cache->head_dimension == 128 ? (e4m3 ? kv8_attention_simple_kernel<128, true> : kv8_attention_simple_kernel<128, false>)
                                                      : (e4m3 ? kv8_attention_simple_kernel<64, true> : kv8_attention_simple_kernel<64, false>);
    kernel<<<grid, kSimpleThreads, 0, s>>>(a);
    return static_cast<int32_t>(cudaGetLastError());
}
