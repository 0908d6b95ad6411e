// Causal attention over an 8-bit paged cache (q3t_launch_kv8_attention): few new tokens a row.
//
// out = sum_j p_j v_j / sum_j p_j, p_j = exp(scale * q . k_j - max), over the positions up to the token's own; k_j and v_j are codes times the
// scale of their page and head.  A (new token, query head) of a KV head is a column; a warp takes pages of 16 tokens for 8 columns:
//   scores    S^T = K Q^T, mma.sync m16n8k16 in fp16: tokens are rows of A (a row's 16-byte loads give whole fragments once the
//             contraction index is permuted alike in Q), columns those of B
//   weights   w_j = exp2(s_j * key scale + log2(value scale) - reference): the value's scale is an addend of the exponent, so that
//             w_j is the weight of the CODE, never large, whatever the scales' sizes; p_j = w_j / value scale for the sum
//   output    O^T += V^T W^T: dims are rows of A (bytes of two tokens interleaved), the weights become B by movmatrix
// Codes become fp16 exactly (int8: the byte behind 0x64 reads 1024 + it; e4m3: one conversion for two).  A column's reference is its first
// maximum until a score exceeds it by 2^8, so that outputs are rescaled almost never; weights are kept 2^6 times larger than that
// needs, which leaves fp16 its 11 bits down to 2^-20 of the largest.
//
// The batch's work, groups of 8 pages (one a warp) of every (row, KV head, 8 columns), is cut into as many equal ranges as there are
// CTAs, wherever that falls.  A CTA merges its warps in shared memory; of what is cut every CTA leaves (reference, sum, output)
// and the one with the last ticket folds them in order, so a result depends on the batch's lengths, not on timing.

#include "kv8.cuh"
#include "q3t_kernels.cuh"

#include <climits>

namespace q3t {
namespace {

constexpr int kRowThreads = 256;
constexpr int kRowWarps = kRowThreads / kWarp;         // = pages of a group
constexpr int kRowCtas = 2 * 148;
constexpr int kColumns = 8;
constexpr float kSlack = 8.0f;                         // log2 of how far a score may exceed its column's reference
constexpr float kLift = 6.0f;                          // log2 of the weight at the reference
constexpr int kCounterBytes = (kRowCtas * 4 + 255) / 256 * 256;

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
    void* scratch;
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
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// D += A (16 x 16, fp16) * B (16 x 8); fragments as in attention.cu
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// an 8 x 8 tile of fp16 across the warp, rows for columns
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
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

__device__ __forceinline__ int4 load16(const uint8_t* p) {
    int4 v;
    asm volatile("ld.global.L1::no_allocate.v4.s32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// What a row asks of the kernel
struct RowWork {
    RowSpan span;
    int last;          // tokens that some new token of the row sees
    int blocks;        // of 8 columns
    int groups;        // of 8 pages, at least one: rows that see nothing have zeros to write
};
__device__ __forceinline__ RowWork row_work(const Kv8AttentionArgs& a, int row, int group) {
    RowWork w;
    w.span = row_span(a.starts, a.lengths, row, a.tokens, a.most, a.max_sequence);
    w.last = min(max(w.span.base + w.span.count, 0), a.max_sequence);
    w.blocks = (w.span.count * group + kColumns - 1) / kColumns;
    w.groups = max(1, (w.last + kRowWarps * kPageTokens - 1) / (kRowWarps * kPageTokens));
    return w;
}

template <int HD, bool E4M3>
__global__ void __launch_bounds__(kRowThreads, 2) kv8_rows_kernel(const Kv8AttentionArgs a) {
    constexpr int kParts = HD / 64;                    // 16-byte pieces of a key that a lane holds
    constexpr int kTiles = HD / 16;                    // of 16 dims
    constexpr int kWords = HD / 32;                    // of a value's dims that a lane holds
    constexpr int kPitch = HD + 4;
    extern __shared__ long long before[];              // [rows]: units of the rows up to each
    __shared__ float part[kRowWarps][kColumns][kPitch];
    __shared__ float tops[kRowWarps][kColumns], totals[kRowWarps][kColumns];
    __shared__ float fold_scale[kRowCtas][kColumns];
    __shared__ long long scan[kRowWarps];
    __shared__ int ticket;
    const int tid = threadIdx.x, lane = tid % kWarp, warp = __shfl_sync(0xffffffffu, tid / kWarp, 0);
    const int g = lane >> 2, q4 = lane & 3;
    const int heads = a.cache.heads, group = a.query_heads / heads;

    // ---- the batch's units, as prefix sums over the rows; the first CTA counts what lies outside the host's bounds
    long long sum = 0;
    for (int first = 0; first < a.rows; first += kRowThreads) {
        const int row = first + tid;
        long long mine = 0;
        if (row < a.rows) {
            const RowWork w = row_work(a, row, group);
            mine = (long long)w.blocks * heads * w.groups;
            if (w.span.cut && blockIdx.x == 0) atomicAdd(&g_kv8_range_errors, 1u);
        }
#pragma unroll
        for (int o = 1; o < kWarp; o <<= 1) {
            const long long other = __shfl_up_sync(0xffffffffu, mine, o);
            if (lane >= o) mine += other;
        }
        if (lane == kWarp - 1) scan[warp] = mine;
        __syncthreads();
        for (int w = 0; w < warp; ++w) mine += scan[w];
        if (row < a.rows) before[row] = sum + mine;
        for (int w = 0; w < kRowWarps; ++w) sum += scan[w];
        __syncthreads();
    }
    const long long units = sum;
    const int ctas = (int)min((long long)gridDim.x, units);
    if ((int)blockIdx.x >= ctas) return;
    long long unit = units * blockIdx.x / ctas;
    const long long unit_first = unit, unit_end = units * (blockIdx.x + 1) / ctas;
    int row;
    {
        int low = 0, high = a.rows - 1;
        while (low < high) {
            const int middle = (low + high) >> 1;
            if (before[middle] > unit) high = middle;
            else low = middle + 1;
        }
        row = low;
    }

    bool waited = false;
    while (unit < unit_end) {
        while (before[row] <= unit) ++row;
        const RowWork w = row_work(a, row, group);
        const long long in_row = unit - (row > 0 ? before[row - 1] : 0);
        const int segment = (int)(in_row / w.groups);              // (KV head, block of columns)
        const int group_first = (int)(in_row - (long long)segment * w.groups);
        const int group_end = (int)min((long long)w.groups, group_first + (unit_end - unit));
        const int kv_head = segment / w.blocks, block = segment - kv_head * w.blocks;
        const int columns = min(kColumns, w.span.count * group - block * kColumns);

        // ---- queries: this lane's column and dims, to fp16 by a power of two that brings the largest to 2^7..2^8
        uint32_t qf[kParts][4][2];
        float column_scale;
        int column_seen;
        {
            const int column = block * kColumns + g;
            const bool real = g < columns;
            const int i = real ? column / group : 0;
            const bf16* q = a.query + (size_t)(w.span.first + i) * a.query_stride + (size_t)(kv_head * group + column % group) * HD + q4 * 16;
            int4 raw[kParts][2];
            uint32_t most = 0u;
#pragma unroll
            for (int j = 0; j < kParts; ++j) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    raw[j][h] = real ? *reinterpret_cast<const int4*>(q + 64 * j + 8 * h) : make_int4(0, 0, 0, 0);
                    const uint32_t x[4] = {(uint32_t)raw[j][h].x, (uint32_t)raw[j][h].y, (uint32_t)raw[j][h].z, (uint32_t)raw[j][h].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) most = __vmaxu2(most, x[e] & 0x7fff7fffu);
                }
            }
            most = max(most & 0xffffu, most >> 16);
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
            const int shift = min(134 - (int)min(most >> 7, 254u), 127);
            const float up = ldexpf(1.0f, shift);
            column_scale = ldexpf(a.scale * 1.4426950408889634f, -shift);
            column_seen = real ? min(max(w.span.base + i + 1, 0), a.max_sequence) : 0;
#pragma unroll
            for (int j = 0; j < kParts; ++j) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t x[4] = {(uint32_t)raw[j][h].x, (uint32_t)raw[j][h].y, (uint32_t)raw[j][h].z, (uint32_t)raw[j][h].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) qf[j][2 * h + e / 2][e & 1] = pack_half2(bf_lo(x[e]) * up, bf_hi(x[e]) * up);
                }
            }
        }
        // of the columns whose scores this lane gets
        const float scale0 = __shfl_sync(0xffffffffu, column_scale, 8 * q4), scale1 = __shfl_sync(0xffffffffu, column_scale, 8 * q4 + 4);
        const int seen0 = __shfl_sync(0xffffffffu, column_seen, 8 * q4), seen1 = __shfl_sync(0xffffffffu, column_seen, 8 * q4 + 4);

        float o[kTiles][4];
#pragma unroll
        for (int t = 0; t < kTiles; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.0f;
        float top0 = -INFINITY, top1 = -INFINITY, sum0 = 0.0f, sum1 = 0.0f;

        // ---- this warp's pages: 8 g + warp; their ids a lane each, 32 at a time
        const int* const ids_at = a.table + (size_t)row * a.table_stride + warp;
        const int pages_end = (w.last + kPageTokens - 1) / kPageTokens;
        auto ids_from = [&](int first) {
            const int page = (first + lane) * kRowWarps + warp;
            return first + lane < group_end && page < pages_end ? ids_at[(size_t)(first + lane) * kRowWarps] : -1;
        };
        int4 kr[kParts][2], vr[4];
        float key_scale, value_scale;
        const size_t k_offset = (size_t)kv_head * (kPageTokens * HD) + g * HD + q4 * 16;
        const size_t v_offset = (size_t)kv_head * (kPageTokens * HD) + 2 * q4 * HD + g * (HD / 8);
        auto load_keys = [&](int id) {
            const uint8_t* k = a.cache.k + (long long)id * a.cache.page_stride + k_offset;
#pragma unroll
            for (int j = 0; j < kParts; ++j) {
                kr[j][0] = load16(k + 64 * j);
                kr[j][1] = load16(k + 64 * j + 8 * HD);
            }
            key_scale = a.cache.k_scales[(long long)id * a.cache.scale_stride + kv_head];
        };
        auto load_values = [&](int id) {
            const uint8_t* v = a.cache.v + (long long)id * a.cache.page_stride + v_offset;
            // tokens 2 q4, + 1, + 8, + 9
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const uint8_t* at = v + ((t & 1) + (t >> 1) * 8) * HD;
                if (HD == 128) {
                    vr[t] = load16(at);
                } else {
                    const int2 half = *reinterpret_cast<const int2*>(at);
                    vr[t] = make_int4(half.x, half.y, 0, 0);
                }
            }
            value_scale = a.cache.v_scales[(long long)id * a.cache.scale_stride + kv_head];
        };
        int ids = ids_from(group_first);
        int raw_id = __shfl_sync(0xffffffffu, ids, 0);
        // (a page that is not there is read as page 0 and masked)
        auto usable = [&](int id) { return id >= 0 && id < a.cache.pages; };
        const bool any = group_first * kRowWarps + warp < pages_end;
        if (any) {
            load_keys(usable(raw_id) ? raw_id : 0);
            load_values(usable(raw_id) ? raw_id : 0);
        }
        for (int gr = group_first; gr < group_end; ++gr) {
            const int page = gr * kRowWarps + warp;
            if (page >= pages_end) break;
            const bool there = usable(raw_id);
            if (!there && segment == 0 && lane == 0) atomicAdd(&g_kv8_page_errors, 1u);
            const int next = gr + 1 - group_first;
            if ((next & 31) == 0) ids = ids_from(gr + 1);
            const int next_raw = __shfl_sync(0xffffffffu, ids, next & 31);
            const int next_id = usable(next_raw) ? next_raw : 0;
            const bool more = gr + 1 < group_end && page + kRowWarps < pages_end;

            // ---- scores
            float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < kParts; ++j) {
                const uint32_t x[4] = {(uint32_t)kr[j][0].x, (uint32_t)kr[j][0].y, (uint32_t)kr[j][0].z, (uint32_t)kr[j][0].w};
                const uint32_t y[4] = {(uint32_t)kr[j][1].x, (uint32_t)kr[j][1].y, (uint32_t)kr[j][1].z, (uint32_t)kr[j][1].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t a0, a1, a2, a3;
                    codes_to_half<E4M3>(x[e], a0, a2);
                    codes_to_half<E4M3>(y[e], a1, a3);
                    mma_f16(s, a0, a1, a2, a3, qf[j][e][0], qf[j][e][1]);
                }
            }
            const float ks = key_scale, vs = fmaxf(value_scale, kKv8SmallestScale);
            if (more) load_keys(next_id);
            // ---- weights of the codes
            const float lv = log2_fast(vs), f0 = ks * scale0, f1 = ks * scale1;
            const int t_low = page * kPageTokens + g, t_high = t_low + 8;
            s[0] = there && t_low < seen0 ? fmaf(s[0], f0, lv) : -INFINITY;
            s[1] = there && t_low < seen1 ? fmaf(s[1], f1, lv) : -INFINITY;
            s[2] = there && t_high < seen0 ? fmaf(s[2], f0, lv) : -INFINITY;
            s[3] = there && t_high < seen1 ? fmaf(s[3], f1, lv) : -INFINITY;
            float m0 = fmaxf(s[0], s[2]), m1 = fmaxf(s[1], s[3]);
            if (__any_sync(0xffffffffu, m0 > top0 + kSlack || m1 > top1 + kSlack)) {
#pragma unroll
                for (int x = 4; x < kWarp; x <<= 1) {
                    m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, x));
                    m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, x));
                }
                const float keep0 = m0 > top0 + kSlack ? exp2_ftz(top0 - m0) : 1.0f;
                const float keep1 = m1 > top1 + kSlack ? exp2_ftz(top1 - m1) : 1.0f;
                top0 = m0 > top0 + kSlack ? m0 : top0;
                top1 = m1 > top1 + kSlack ? m1 : top1;
                sum0 *= keep0;
                sum1 *= keep1;
#pragma unroll
                for (int t = 0; t < kTiles; ++t) {
                    o[t][0] *= keep0;
                    o[t][1] *= keep1;
                    o[t][2] *= keep0;
                    o[t][3] *= keep1;
                }
            }
            // (nothing but -inf so far: weights of zero)
            const float r0 = top0 == -INFINITY ? 0.0f : top0 - kLift, r1 = top1 == -INFINITY ? 0.0f : top1 - kLift;
            const float w0 = exp2_ftz(s[0] - r0), w1 = exp2_ftz(s[1] - r1), w2 = exp2_ftz(s[2] - r0), w3 = exp2_ftz(s[3] - r1);
            const float inverse = __frcp_rn(vs);
            sum0 = fmaf(w0 + w2, inverse, sum0);
            sum1 = fmaf(w1 + w3, inverse, sum1);
            const uint32_t b0 = transpose8(pack_half2(w0, w1)), b1 = transpose8(pack_half2(w2, w3));
            // ---- output; what lies behind the row's last token may read as NaN, which no weight of zero removes
            if (E4M3 && (page + 1) * kPageTokens > w.last) {
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    if (page * kPageTokens + 2 * q4 + (t & 1) + (t >> 1) * 8 >= w.last) vr[t] = make_int4(0, 0, 0, 0);
                }
            }
            if (E4M3 && !there) vr[0] = vr[1] = vr[2] = vr[3] = make_int4(0, 0, 0, 0);
#pragma unroll
            for (int e = 0; e < kWords; ++e) {
                const auto word = [&](const int4& v) { return (uint32_t)(e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w); };
                // bytes of two tokens side by side, dims 4 e, + 1 and 4 e + 2, + 3 of this lane
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t a0, a1, a2, a3;
                    codes_to_half<E4M3>(__byte_perm(word(vr[0]), word(vr[1]), h == 0 ? 0x5140 : 0x7362), a0, a1);
                    codes_to_half<E4M3>(__byte_perm(word(vr[2]), word(vr[3]), h == 0 ? 0x5140 : 0x7362), a2, a3);
                    mma_f16(o[2 * e + h], a0, a1, a2, a3, b0, b1);
                }
            }
            if (more) load_values(next_id);
            raw_id = next_raw;
        }

        // ---- the CTA's warps together
#pragma unroll
        for (int x = 4; x < kWarp; x <<= 1) {
            sum0 += __shfl_xor_sync(0xffffffffu, sum0, x);
            sum1 += __shfl_xor_sync(0xffffffffu, sum1, x);
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            if (2 * q4 + c < columns) {
                float* const at = &part[warp][2 * q4 + c][g * (HD / 8)];
#pragma unroll
                for (int t = 0; t < kTiles; t += 2) {
                    *reinterpret_cast<float4*>(at + 2 * t) = make_float4(o[t][c], o[t][c + 2], o[t + 1][c], o[t + 1][c + 2]);
                }
            }
        }
        if (g == 0) {
            tops[warp][2 * q4] = top0;
            tops[warp][2 * q4 + 1] = top1;
            totals[warp][2 * q4] = sum0;
            totals[warp][2 * q4 + 1] = sum1;
        }
        __syncthreads();
        const bool whole = group_first == 0 && group_end == w.groups;
        float* const pieces = reinterpret_cast<float*>(static_cast<char*>(a.scratch) + kCounterBytes);
        constexpr int kPiece = kColumns * (HD + 2);                // [column][HD], then tops, then sums
        float* const piece = pieces + (size_t)(2 * blockIdx.x + (unit == unit_first ? 0 : 1)) * kPiece;
        auto write = [&](int column, int d, float value) {
            const int c = block * kColumns + column, i = c / group;
            const size_t token = w.span.first + i, at = (size_t)(kv_head * group + c % group) * HD + d;
            a.out[token * a.out_stride + at] = f2bf(value);
            if (a.out32 != nullptr) a.out32[token * a.query_heads * HD + at] = value;
        };
        for (int x = tid; x < columns * HD; x += kRowThreads) {
            const int column = x / HD, d = x % HD;
            float top = tops[0][column], total = 0.0f, value = 0.0f;
#pragma unroll
            for (int v = 1; v < kRowWarps; ++v) top = fmaxf(top, tops[v][column]);
#pragma unroll
            for (int v = 0; v < kRowWarps; ++v) {
                const float f = tops[v][column] == -INFINITY ? 0.0f : exp2_ftz(tops[v][column] - top);
                total += f * totals[v][column];
                value += f * part[v][column][d];
            }
            if (whole) {
                write(column, d, total == 0.0f ? 0.0f : value / total);
            } else {
                piece[column * HD + d] = value;
                if (d == 0) {
                    piece[kColumns * HD + column] = top;
                    piece[kColumns * (HD + 1) + column] = total;
                }
            }
        }
        if (!whole) {
            // ---- of the CTAs that share the segment the last one folds what they left
            const long long start = unit - group_first, end = start + w.groups - 1;
            auto owner = [&](long long u) { return (int)(((u + 1) * ctas - 1) / units); };
            const int first_cta = owner(start), last_cta = owner(end), count = last_cta - first_cta + 1;
            if (!waited) {
                pdl_wait();                                        // the counters are zero
                waited = true;
            }
            __threadfence();
            __syncthreads();
            if (tid == 0) ticket = (int)atomicAdd(static_cast<unsigned int*>(a.scratch) + first_cta, 1u);
            __syncthreads();
            if (ticket == count - 1) {
                __threadfence();
                // the first CTA's range may begin before the segment: its second piece then
                const int lead = units * first_cta / ctas == start ? 0 : 1;
                auto piece_of = [&](int n) { return pieces + (size_t)(2 * (first_cta + n) + (n == 0 ? lead : 0)) * kPiece; };
                for (int x = tid; x < count * kColumns; x += kRowThreads) {
                    if (x % kColumns < columns) fold_scale[x / kColumns][x % kColumns] = __ldcg(piece_of(x / kColumns) + kColumns * HD + x % kColumns);
                }
                __syncthreads();
                for (int x = tid; x < columns * HD; x += kRowThreads) {
                    const int column = x / HD, d = x % HD;
                    float top = -INFINITY, total = 0.0f, value = 0.0f;
                    for (int n = 0; n < count; ++n) top = fmaxf(top, fold_scale[n][column]);
#pragma unroll 4
                    for (int n = 0; n < count; ++n) {
                        const float f = fold_scale[n][column] == -INFINITY ? 0.0f : exp2_ftz(fold_scale[n][column] - top);
                        total += f * __ldcg(piece_of(n) + kColumns * (HD + 1) + column);
                        value += f * __ldcg(piece_of(n) + column * HD + d);
                    }
                    write(column, d, total == 0.0f ? 0.0f : value / total);
                }
            }
        }
        __syncthreads();
        unit += group_end - group_first;
    }
    if (!waited) pdl_wait();
    pdl_trigger();
}

template <int HD, bool E4M3>
cudaError_t launch_rows(const Kv8AttentionArgs& a, cudaStream_t stream) {
    static std::atomic<unsigned long long> allowed{0};
    cudaError_t e = kv8_allow_smem(allowed, kv8_rows_kernel<HD, E4M3>, Q3T_MAX_TABLE_ROWS * (int)sizeof(long long));
    if (e == cudaSuccess) e = launch_zero_counters(static_cast<unsigned int*>(a.scratch), kRowCtas, stream);
    if (e != cudaSuccess) return e;
    return launch_pdl(kv8_rows_kernel<HD, E4M3>, dim3(kRowCtas), dim3(kRowThreads), (size_t)a.rows * sizeof(long long), stream, a);
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
    if (!q3t::attention_args(desc, &a)) return 0;
    return q3t::kCounterBytes + (size_t)q3t::kRowCtas * 2 * q3t::kColumns * (desc->cache->head_dimension + 2) * sizeof(float);
}

extern "C" int32_t q3t_launch_kv8_attention(const Q3tKv8AttentionDesc* desc, void* stream) {
    using namespace q3t;
    Kv8AttentionArgs a;
    if (!attention_args(desc, &a) || desc->scratch == nullptr || reinterpret_cast<uintptr_t>(desc->scratch) % 16 != 0
        || desc->scratch_bytes < q3t_kv8_attention_scratch_bytes(desc)) {
        return cudaErrorInvalidValue;
    }
    if (a.most == 0) return cudaSuccess;
    a.scratch = desc->scratch;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool e4m3 = desc->cache->format == Q3T_KV8_E4M3;
    if (desc->cache->head_dimension == 128) return static_cast<int32_t>(e4m3 ? launch_rows<128, true>(a, s) : launch_rows<128, false>(a, s));
    return static_cast<int32_t>(e4m3 ? launch_rows<64, true>(a, s) : launch_rows<64, false>(a, s));
}
