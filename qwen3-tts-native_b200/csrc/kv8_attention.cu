// Causal attention over an 8-bit paged cache (q3t_launch_kv8_attention): rows of few new tokens.  kv8_prompt.cu has the others.
//
// out = sum_j p_j v_j / sum_j p_j, p_j = exp(scale * q . k_j - max), over the positions up to the token's own; k_j and v_j are codes times the
// scale of their page and head.  A (new token, query head) of a KV head is a column; a warp takes pages of 16 tokens for 8 or 16 columns:
//   scores    S^T = K Q^T, mma.sync m16n8k16 in fp16: tokens are rows of A (a row's 16-byte loads give whole fragments once the
//             contraction index is permuted alike in Q), columns those of B
//   weights   w_j = exp2(s_j * key scale + log2(value scale) - reference): the value's scale is an addend of the exponent, so that
//             w_j is the weight of the CODE, never large, whatever the scales' sizes; p_j = w_j / value scale for the sum
//   output    O^T += V^T W^T: dims are rows of A (bytes of two tokens interleaved), the weights become B by movmatrix
// Codes become fp16 exactly (int8: the byte behind 0x64 reads 1024 + it; e4m3: one conversion for two).  A column's reference is its first
// maximum until a score exceeds it by 2^8, so that outputs are rescaled almost never; weights are kept 2^6 times larger than that
// needs, which leaves fp16 its 11 bits down to 2^-20 of the largest.
//
// Where segments, (row, KV head, block of 8 columns), are few or short, each is a CTA's or a cluster's (kv8_few_rows_kernel).  Else the
// batch's work, the pages of every segment, is cut into as many equal ranges as there are warps, wherever that falls
// (kv8_rows_kernel).  A warp writes what it has whole; what is cut is merged by the CTA in shared memory, and of what its range cuts
// the CTA leaves (reference, sum, output) and the one with the last ticket folds them in order, so a result depends on
// the batch's lengths, not on timing.
//
// What bounds it: one row, latencies one behind the other (3,000 tokens, 8 heads of 128: 7.1 us); a full batch memory (64 rows of 64 to 2,048 tokens,
// 140 MB: 31 us, of which 21 are memory's; 7 rows of 90,000 to 131,072, 4 heads, 804 MB: 133 us, 6.0 TB/s); rows of several tokens the conversions
// and products of 4 warps a scheduler that each wait for their next page (23 drafts of five, heads of 64, 48 MB: 23 us).  (Times here and below are
// those of the same call 20 times in a graph; on inputs that change from call to call these four take 8.2, 33, 143 and 24 us.)

#include "kv8.cuh"
#include "q3t_kernels.cuh"
#include "q3t_tcgen05.cuh"

#include <climits>

namespace q3t {

// kv8_prompt.cu.  As much as any launch of rows no longer may need
size_t kv8_prompt_scratch_bytes(int max_sequence, int head_dim);
cudaError_t launch_kv8_prompts(const Kv8AttentionArgs& a, int head_dim, bool e4m3, cudaStream_t stream);

namespace {

constexpr int kRowThreads = 256;
constexpr int kRowWarps = kRowThreads / kWarp;
constexpr int kRowCtas = 2 * 148;
constexpr int kTileColumns = 8;                        // of a product
constexpr int kStartUnits = 2;                         // what the start of a segment counts for in the cut, in pages (1 to 3: the same; 4: 2 % more)
constexpr int kClusterCtas = 8;                        // the most of a segment
// Clusters as large as lets all segments' CTAs run at once (256 of 296 places: clusters leave some), and not so large that warps have
// less than half a page; up to 1,024 tokens a CTA.  One token a row, 8 KV heads of 128, clusters / ranges in us: 1 row of 64 tokens 4.1 / 8.6, of
// 8,192 11.4 / 12.7, of 16,384 18.6 / 14.9; 8 rows of 4,096 15.6 / 18.5; 16 of 2,048 15.3 / 18.7, of 4,096 27.4 / 29.7; 32 of 1,024 15.2 / 20.2, of 2,048
// 28.7 / 30.7.  (Rows of one length, which suits the clusters: others leave some idle where ranges are even.  Hence the bound on the near side.)
// Short rows also in two rounds: 64 rows of 64 8.1 / 11.1, of 256 12.3 / 14.7, of 512 17.7 / 19.8, of 1 to 512 13.7 / 15.2, of 1,024 31.5 / 30.7.
// One row has so many segments where it is a prompt, which kv8_prompt.cu takes in one launch: as soon where some SM here has a fourth CTA.  Clusters /
// prompts, 16 query heads on 8 of 128, from nothing: 136 tokens (272 CTAs) 6.3 / 9.9, 160 9.8 / 9.8, 216 (432) 10.6 / 10.5, 232 (464) 12.3 / 10.5, 256
// (512) 12.7 / 10.8; over 512: 136 9.5 / 14.4, 216 14.8 / 14.4, 232 17.3 / 14.4, 256 17.5 / 14.2.  (Heads of 64, 256 tokens: 9.7 / 8.9 and 12.7 / 11.7.)  Two
// rows of 128 tokens (512 CTAs), behind the launches for rows that are none: 8.8 / 11.4.
constexpr int kFewCtas = 256, kOnePromptCtas = 3 * 148, kFewTokens = 1024, kFewest = 64;
// Rows of more columns than this are kv8_prompt.cu's, which takes 64 tokens for 128 columns in the time it takes them for one.  64 rows over 2,048
// tokens, here / there in us: 32 columns 127 / 132, 48 167 / 132; 16 rows: 32 36 / 37, 48 45 / 37.
constexpr int kRowColumns = 32;
// But too few of them leave SMs idle there: they stay here while (query heads x new tokens x tokens seen) is below 2^23, unless even the longest
// context takes no time there.  One row, 8 KV heads, the ranges / there: over 16,384 48 columns 34 / 40, 64 (2^23) 40 / 40, 256 111 / 51; over
// 2,048 256 columns 27 / 30, 512 (2^23) 39 / 31; over 1,024 512 columns 27 / 21; over 256 512 columns 16 / 11.  A row alone that goes there is the only
// one, so that nothing is launched here (a prompt of 1,500 tokens 27.5 us, with two launches for rows that are not there 29.2).
constexpr long long kPromptWork = 1 << 23;
constexpr int kShort = 1024;
constexpr int kCounterBytes = (kRowCtas * 4 + 255) / 256 * 256;

__device__ unsigned int g_kv8_range_errors = 0;
__device__ unsigned int g_kv8_page_errors = 0;

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
__device__ __forceinline__ int4 load16(const uint8_t* p) {
    int4 v;
    asm volatile("ld.global.L1::no_allocate.v4.s32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// of another CTA's shared memory
__device__ __forceinline__ float2 peer_float2(uint32_t at) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ float4 peer_float4(uint32_t at) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}

// What a row asks of the kernel
struct RowWork {
    RowSpan span;
    int last;          // tokens that some new token of the row sees
    int blocks;        // of 8 or 16 columns; none where the row is kv8_prompt.cu's
    int pages;         // at least one: rows that see nothing have zeros to write
};
__device__ __forceinline__ RowWork row_work(const Kv8AttentionArgs& a, int row, int group, int block_columns) {
    RowWork w;
    w.span = row_span(a.starts, a.lengths, row, a.tokens, a.most, a.max_sequence);
    w.last = min(max(w.span.base + w.span.count, 0), a.max_sequence);
    w.blocks = w.span.count * group > a.row_columns ? 0 : (w.span.count * group + block_columns - 1) / block_columns;
    w.pages = max(1, (w.last + kPageTokens - 1) / kPageTokens);
    return w;
}

// A segment, (row, KV head, block of columns), of which a warp takes some pages
struct Segment {
    int row, kv_head;
    int column;        // of the row and KV head: the first
    int columns;
    bool counts;       // its pages that are not there
};

// 8 dims of a column of a row and KV head, from where its new tokens begin
template <int HD>
__device__ __forceinline__ void write8(const Kv8AttentionArgs& a, int first, int kv_head, int column, int d, const float (&v)[8]) {
    const int group = a.query_heads / a.cache.heads, i = column / group;
    const size_t token = first + i, at = (size_t)(kv_head * group + column - i * group) * HD + d;
    __nv_bfloat162 x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
    *reinterpret_cast<int4*>(a.out + token * a.out_stride + at) = *reinterpret_cast<const int4*>(x);
    if (a.out32 != nullptr) {
        float* const to = a.out32 + token * a.query_heads * HD + at;
        *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(to + 4) = make_float4(v[4], v[5], v[6], v[7]);
    }
}

// A warp's way through pages of a segment.  Lane 4 g + q4 holds dims g * HD / 8 and on of columns 2 q4 and + 1 of each tile.
template <int HD, bool E4M3, int TILES>
struct Walk {
    static constexpr int kColumns = TILES * kTileColumns;
    static constexpr int kParts = HD / 64;             // 16-byte pieces of a key that a lane holds
    static constexpr int kTiles = HD / 16;             // of 16 dims
    static constexpr int kWords = HD / 32;             // of a value's dims that a lane holds
    static constexpr int kPitch = HD + 4;              // of a column of a piece: its output, then reference and sum
    static constexpr int kPiece = kColumns * kPitch;
    float o[TILES][kTiles][4], top[TILES][2], sum_of[TILES][2];

    __device__ __forceinline__ Walk() {
#pragma unroll
        for (int n = 0; n < TILES; ++n) {
            top[n][0] = top[n][1] = -INFINITY;
            sum_of[n][0] = sum_of[n][1] = 0.0f;
#pragma unroll
            for (int t = 0; t < kTiles; ++t) o[n][t][0] = o[n][t][1] = o[n][t][2] = o[n][t][3] = 0.0f;
        }
    }

    // pages page_first .. page_end - 1, at least one.  AHEAD: the page after the next one is called into the L2, a line a lane, where a warp
    // walks many of 4 KB (64 rows of 8,192 tokens: 169 us, without 176.5; heads of 64, which wait for instructions: 6 % longer with it)
    template <bool AHEAD>
    __device__ __forceinline__ void run(const Kv8AttentionArgs& a, const RowWork& w, const Segment& of, int page_first, int page_end) {
        const int row = of.row, kv_head = of.kv_head, columns = of.columns;
        const bool counts = of.counts;
        // ---- pages: their ids a lane each, 32 at a time (one that is not there is read as page 0 and masked)
        const int lane = threadIdx.x % kWarp, g = lane >> 2, q4 = lane & 3, group = a.query_heads / a.cache.heads;
        const int* const ids_at = a.table + (size_t)row * a.table_stride;
        auto usable = [&](int id) { return id >= 0 && id < a.cache.pages; };
        auto ids_from = [&](int first) { return first + lane < page_end && (first + lane) * kPageTokens < w.last ? ids_at[first + lane] : -1; };
        int ids = ids_from(page_first);

        // ---- queries: this lane's columns and dims, to fp16 by a power of two that brings the largest to 2^7..2^8
        uint32_t qf[TILES][kParts][4][2];
        float column_scale[TILES];
        int column_seen[TILES];
        int4 raw[TILES][kParts][2];
#pragma unroll
        for (int n = 0; n < TILES; ++n) {
            const int of_block = n * kTileColumns + g, column = of.column + of_block;
            const bool real = of_block < columns;
            const int i = real ? column / group : 0;
            const bf16* q = a.query + (size_t)(w.span.first + i) * a.query_stride + (size_t)(kv_head * group + column % group) * HD + q4 * 16;
#pragma unroll
            for (int j = 0; j < kParts; ++j) {
#pragma unroll
                for (int h = 0; h < 2; ++h) raw[n][j][h] = real ? *reinterpret_cast<const int4*>(q + 64 * j + 8 * h) : make_int4(0, 0, 0, 0);
            }
            column_seen[n] = real ? min(max(w.span.base + i + 1, 0), a.max_sequence) : 0;
        }
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
        int raw_id = __shfl_sync(0xffffffffu, ids, 0);
        load_keys(usable(raw_id) ? raw_id : 0);
        load_values(usable(raw_id) ? raw_id : 0);
#pragma unroll
        for (int n = 0; n < TILES; ++n) {
            uint32_t most = 0u;
#pragma unroll
            for (int j = 0; j < kParts; ++j) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t x[4] = {(uint32_t)raw[n][j][h].x, (uint32_t)raw[n][j][h].y, (uint32_t)raw[n][j][h].z, (uint32_t)raw[n][j][h].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) most = __vmaxu2(most, x[e] & 0x7fff7fffu);
                }
            }
            most = max(most & 0xffffu, most >> 16);
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
            const int shift = query_shift(most);
            const float up = power_of_two(shift);
            column_scale[n] = query_back(a.scale * 1.4426950408889634f, shift);
#pragma unroll
            for (int j = 0; j < kParts; ++j) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t x[4] = {(uint32_t)raw[n][j][h].x, (uint32_t)raw[n][j][h].y, (uint32_t)raw[n][j][h].z, (uint32_t)raw[n][j][h].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) qf[n][j][2 * h + e / 2][e & 1] = pack_half2(bf_lo(x[e]) * up, bf_hi(x[e]) * up);
                }
            }
        }
        // of the columns whose scores this lane gets, 2 q4 and + 1 of each tile
        float scale_of[TILES][2];
        int seen[TILES][2];
#pragma unroll
        for (int n = 0; n < TILES; ++n) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                scale_of[n][c] = __shfl_sync(0xffffffffu, column_scale[n], 8 * q4 + 4 * c);
                seen[n][c] = __shfl_sync(0xffffffffu, column_seen[n], 8 * q4 + 4 * c);
            }
        }

        for (int page = page_first; page < page_end; ++page) {
            const bool there = usable(raw_id);
            if (!there && counts && lane == 0 && page * kPageTokens < w.last) atomicAdd(&g_kv8_page_errors, 1u);
            const int next = page + 1 - page_first;
            if ((next & 31) == 0) ids = ids_from(page + 1);
            const int next_raw = __shfl_sync(0xffffffffu, ids, next & 31);
            const int next_id = usable(next_raw) ? next_raw : 0;
            const bool more = page + 1 < page_end;
            if (AHEAD && page + 2 < page_end && (next & 31) != 31) {
                const int ahead = __shfl_sync(0xffffffffu, ids, (next + 1) & 31);
                constexpr int kLines = kPageTokens * HD / 128;
                const uint8_t* const plane = lane < kLines ? a.cache.k : a.cache.v;
                if (lane < 2 * kLines && usable(ahead)) {
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(plane + (long long)ahead * a.cache.page_stride + (size_t)kv_head * (kPageTokens * HD) + lane % kLines * 128));
                }
            }

            // ---- scores
            float s[TILES][4];
#pragma unroll
            for (int n = 0; n < TILES; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
#pragma unroll
            for (int j = 0; j < kParts; ++j) {
                const uint32_t x[4] = {(uint32_t)kr[j][0].x, (uint32_t)kr[j][0].y, (uint32_t)kr[j][0].z, (uint32_t)kr[j][0].w};
                const uint32_t y[4] = {(uint32_t)kr[j][1].x, (uint32_t)kr[j][1].y, (uint32_t)kr[j][1].z, (uint32_t)kr[j][1].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t a0, a1, a2, a3;
                    codes_to_half<E4M3>(x[e], a0, a2);
                    codes_to_half<E4M3>(y[e], a1, a3);
#pragma unroll
                    for (int n = 0; n < TILES; ++n) mma_f16(s[n], a0, a1, a2, a3, qf[n][j][e][0], qf[n][j][e][1]);
                }
            }
            const float ks = key_scale, vs = fmaxf(value_scale, kKv8LeastValueScale);
            const float back = fminf(value_scale * (1.0f / kKv8LeastValueScale), 1.0f);
            if (more) load_keys(next_id);
            // ---- weights of the codes
            const float lv = log2_fast(vs), inverse = reciprocal_fast(vs);
            const int t_low = page * kPageTokens + g, t_high = t_low + 8;
            uint32_t b0[TILES], b1[TILES];
#pragma unroll
            for (int n = 0; n < TILES; ++n) {
                float m[2];
                bool moves = false;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const float f = ks * scale_of[n][c];
                    s[n][c] = there && t_low < seen[n][c] ? fmaf(s[n][c], f, lv) : -INFINITY;
                    s[n][2 + c] = there && t_high < seen[n][c] ? fmaf(s[n][2 + c], f, lv) : -INFINITY;
                    m[c] = fmaxf(s[n][c], s[n][2 + c]);
                    moves |= m[c] > top[n][c] + kKv8Slack;
                }
                if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
#pragma unroll
                        for (int x = 4; x < kWarp; x <<= 1) m[c] = fmaxf(m[c], __shfl_xor_sync(0xffffffffu, m[c], x));
                        const bool up = m[c] > top[n][c] + kKv8Slack;
                        const float keep = up ? exp2_ftz(top[n][c] - m[c]) : 1.0f;
                        top[n][c] = up ? m[c] : top[n][c];
                        sum_of[n][c] *= keep;
#pragma unroll
                        for (int t = 0; t < kTiles; ++t) {
                            o[n][t][c] *= keep;
                            o[n][t][2 + c] *= keep;
                        }
                    }
                }
                float low[2], high[2];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    // (nothing but -inf so far: weights of zero)
                    const float reference = top[n][c] == -INFINITY ? 0.0f : top[n][c] - kKv8Lift;
                    low[c] = exp2_ftz(s[n][c] - reference);
                    high[c] = exp2_ftz(s[n][2 + c] - reference);
                    sum_of[n][c] = fmaf(low[c] + high[c], inverse, sum_of[n][c]);
                }
                if (back != 1.0f) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        low[c] *= back;
                        high[c] *= back;
                    }
                }
                b0[n] = transpose8(pack_half2(low[0], low[1]));
                b1[n] = transpose8(pack_half2(high[0], high[1]));
            }
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
#pragma unroll
                    for (int n = 0; n < TILES; ++n) mma_f16(o[n][2 * e + h], a0, a1, a2, a3, b0[n], b1[n]);
                }
            }
            if (more) load_values(next_id);
            raw_id = next_raw;
        }
    }

    // into shared memory
    __device__ __forceinline__ void keep(float* piece, int columns) const {
        const int lane = threadIdx.x % kWarp, g = lane >> 2, q4 = lane & 3;
#pragma unroll
        for (int n = 0; n < TILES; ++n) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float total = sum_of[n][c];
#pragma unroll
                for (int x = 4; x < kWarp; x <<= 1) total += __shfl_xor_sync(0xffffffffu, total, x);
                const int column = n * kTileColumns + 2 * q4 + c;
                if (column >= columns) continue;
                float* const at = piece + column * kPitch;
#pragma unroll
                for (int t = 0; t < kTiles; t += 2) {
                    *reinterpret_cast<float4*>(at + g * (HD / 8) + 2 * t) = make_float4(o[n][t][c], o[n][t][c + 2], o[n][t + 1][c], o[n][t + 1][c + 2]);
                }
                if (g == 0) *reinterpret_cast<float2*>(at + HD) = make_float2(top[n][c], total);
            }
        }
    }

    // a whole segment
    __device__ __forceinline__ void write(const Kv8AttentionArgs& a, int first, const Segment& of) const {
        const int lane = threadIdx.x % kWarp, g = lane >> 2, q4 = lane & 3;
#pragma unroll
        for (int n = 0; n < TILES; ++n) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float total = sum_of[n][c];
#pragma unroll
                for (int x = 4; x < kWarp; x <<= 1) total += __shfl_xor_sync(0xffffffffu, total, x);
                const int column = n * kTileColumns + 2 * q4 + c;
                if (column >= of.columns) continue;
                const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
                for (int t = 0; t < kTiles; t += 4) {
                    const float v[8] = {o[n][t][c] * inverse, o[n][t][c + 2] * inverse, o[n][t + 1][c] * inverse, o[n][t + 1][c + 2] * inverse,
                                        o[n][t + 2][c] * inverse, o[n][t + 2][c + 2] * inverse, o[n][t + 3][c] * inverse, o[n][t + 3][c + 2] * inverse};
                    write8<HD>(a, first, of.kv_head, of.column + column, g * (HD / 8) + 2 * t, v);
                }
            }
        }
    }
};

// 64-bit divisions take hundreds of instructions, where a CTA has nothing else to do; most fit 32 bits
__device__ __forceinline__ long long quotient(long long x, long long y) {
    return ((x | y) >> 32) == 0 ? (long long)((unsigned int)x / (unsigned int)y) : x / y;
}
__device__ __forceinline__ long long share_of(long long units, int n, int of) { return quotient(units * n, of); }

// The tickets of the launch behind it, which is let in at once and waits for this one before anything else: it lies in wait on the SMs
// while the launch ahead of both ends
__global__ void kv8_zero_tickets_kernel(unsigned int* tickets) {
    pdl_trigger();
    pdl_wait();
    tickets[threadIdx.x] = 0u;
}

// A part of a segment, (row, KV head, block of columns): whose it is
struct Piece {
    long long start;   // unit of the segment's first page, -1: none
    int pages;         // of the segment
    int first;         // number of the row's first new token
    int kv_head;
    int column;        // of the row and KV head: the segment's first
    int columns;       // of the segment
};

template <int HD, int TILES>
constexpr size_t rows_smem(int rows) {
    return (size_t)rows * sizeof(long long) + (size_t)2 * kRowWarps * TILES * kTileColumns * (HD + 4) * sizeof(float);
}
// CTAs of an SM: a warp of two tiles of columns and heads of 128 holds twice the outputs and queries
template <int HD, int TILES>
constexpr int rows_residency() {
    return HD == 128 && TILES == 2 ? 1 : 2;
}

template <int HD, bool E4M3, int TILES>
__global__ void __launch_bounds__(kRowThreads, rows_residency<HD, TILES>()) kv8_rows_kernel(const Kv8AttentionArgs a) {
    constexpr int kColumns = TILES * kTileColumns, kPitch = Walk<HD, E4M3, TILES>::kPitch, kPiece = Walk<HD, E4M3, TILES>::kPiece;
    extern __shared__ __align__(16) unsigned char smem[];
    float* const parts = reinterpret_cast<float*>(smem);                                    // [warp][2] pieces
    long long* const before = reinterpret_cast<long long*>(parts + 2 * kRowWarps * kPiece);  // [rows]: units of the rows up to each
    __shared__ Piece held[2 * kRowWarps];
    __shared__ long long scan[kRowWarps];
    __shared__ int folds[2];                           // of the segments that go beyond the CTA at its start and its end: the piece, if it is up to this CTA
    const int tid = threadIdx.x, lane = tid % kWarp, warp = __shfl_sync(0xffffffffu, tid / kWarp, 0);
    const int heads = a.cache.heads, group = a.query_heads / heads;

    pdl_wait();
    if (a.prompts) pdl_trigger();                      // (they may run beside this one)
    // ---- the batch's units (of a segment its start, then its pages), as prefix sums over the rows; the first CTA counts what lies outside the host's bounds
    long long sum = 0;
    for (int first = 0; first < a.rows; first += kRowThreads) {
        const int row = first + tid;
        long long mine = 0;
        if (row < a.rows) {
            const RowWork w = row_work(a, row, group, kColumns);
            mine = (long long)w.blocks * heads * (w.pages + kStartUnits);
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
    const int ctas = (int)min((long long)gridDim.x, (units + kRowWarps - 1) / kRowWarps);
    if ((int)blockIdx.x >= ctas) return;
    const long long cta_first = share_of(units, (int)blockIdx.x, ctas), cta_end = share_of(units, (int)blockIdx.x + 1, ctas);
    long long unit = cta_first + (cta_end - cta_first) * warp / kRowWarps;
    const long long unit_end = cta_first + (cta_end - cta_first) * (warp + 1) / kRowWarps;
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
    if (tid < 2) folds[tid] = -1;
    if (lane < 2) held[2 * warp + lane].start = -1;
    __syncwarp();

    int pieces_held = 0;
    while (unit < unit_end) {
        while (before[row] <= unit) ++row;
        const RowWork w = row_work(a, row, group, kColumns);
        const long long row_first = row > 0 ? before[row - 1] : 0;
        const int segment = (int)quotient(unit - row_first, w.pages + kStartUnits);          // (KV head, block of columns)
        const long long start = row_first + (long long)segment * (w.pages + kStartUnits) + kStartUnits;
        const int page_first = (int)max(unit - start, 0ll);
        const int page_end = (int)min((long long)w.pages, unit_end - start);
        unit = start + w.pages;
        if (page_end <= page_first) continue;
        const int kv_head = segment / w.blocks, block = segment - kv_head * w.blocks;
        const int columns = min(kColumns, w.span.count * group - block * kColumns);

        const Segment of{row, kv_head, block * kColumns, columns, segment == 0};
        Walk<HD, E4M3, TILES> walk;
        walk.template run<HD == 128>(a, w, of, page_first, page_end);
        // ---- whole: written; cut: into shared memory
        if (page_first == 0 && page_end == w.pages) {
            walk.write(a, w.span.first, of);
        } else {
            walk.keep(parts + (size_t)(2 * warp + pieces_held) * kPiece, columns);
            if (lane == 0) held[2 * warp + pieces_held] = Piece{start, w.pages, w.span.first, kv_head, block * kColumns, columns};
            ++pieces_held;
        }
    }
    __syncthreads();

    // ---- pieces of a segment that lie in this CTA stand in order; warps merge them, 32 times 8 dims of its columns each
    float* const left = reinterpret_cast<float*>(static_cast<char*>(a.scratch) + kCounterBytes);
    auto left_by = [&](int cta, int which) { return left + (size_t)(2 * cta + which) * kPiece; };
    // the CTA whose range has a unit
    auto owner = [&](long long u) { return u >= cta_first && u < cta_end ? (int)blockIdx.x : (int)quotient((u + 1) * ctas - 1, units); };
    auto finish = [&](const Piece& p, int column, int d, Merged& v) {
        const float inverse = v.total == 0.0f ? 0.0f : 1.0f / v.total;
#pragma unroll
        for (int e = 0; e < 8; ++e) v.sum[e] *= inverse;
        write8<HD>(a, p.first, p.kv_head, p.column + column, d, v.sum);
    };
    auto put = [&](float* piece, int column, int d, const Merged& v) {
        float* const to = piece + column * kPitch;
        *reinterpret_cast<float4*>(to + d) = make_float4(v.sum[0], v.sum[1], v.sum[2], v.sum[3]);
        *reinterpret_cast<float4*>(to + d + 4) = make_float4(v.sum[4], v.sum[5], v.sum[6], v.sum[7]);
        if (d == 0) *reinterpret_cast<float2*>(to + HD) = make_float2(v.top, v.total);
    };
    auto chunks_of = [](const Piece& p) { return (p.columns * (HD / 8) + kWarp - 1) / kWarp; };
    {
        const long long mine = lane < 2 * kRowWarps ? held[lane].start : -1;
        const unsigned int real = __ballot_sync(0xffffffffu, mine >= 0);
        const unsigned int lower = real & ((1u << lane) - 1u);
        const long long previous = __shfl_sync(0xffffffffu, mine, lower != 0u ? 31 - __clz(lower) : 0);
        unsigned int leads = __ballot_sync(0xffffffffu, mine >= 0 && (lower == 0u || previous != mine));
        for (int n = 0; leads != 0u; ++n) {
            const int first = __ffs(leads) - 1;
            leads &= leads - 1;
            if (n % kRowWarps != warp) continue;
            const unsigned int parts_here = real & ~((1u << first) - 1u) & (leads != 0u ? (leads & -leads) - 1u : ~0u);
            const Piece p = held[first];
            const bool whole = p.start >= cta_first && p.start + p.pages <= cta_end;
            const int which = p.start < cta_first ? 0 : 1;
            float* const to = left_by(blockIdx.x, which);
            for (int x = lane; x < p.columns * (HD / 8); x += kWarp) {
                const int column = x / (HD / 8), d = x % (HD / 8) * 8;
                const float* const at = parts + column * kPitch;
                Merged v;
                for (unsigned int rest = parts_here; rest != 0u; rest &= rest - 1) {
                    const float* const from = at + (__ffs(rest) - 1) * kPiece;
                    v.add(*reinterpret_cast<const float2*>(from + HD), *reinterpret_cast<const float4*>(from + d), *reinterpret_cast<const float4*>(from + d + 4));
                }
                if (whole) {
                    finish(p, column, d, v);
                } else {
                    *reinterpret_cast<float4*>(to + column * kPitch + d) = make_float4(v.sum[0], v.sum[1], v.sum[2], v.sum[3]);
                    *reinterpret_cast<float4*>(to + column * kPitch + d + 4) = make_float4(v.sum[4], v.sum[5], v.sum[6], v.sum[7]);
                    if (d == 0) *reinterpret_cast<float2*>(to + column * kPitch + HD) = make_float2(v.top, v.total);
                }
            }
            if (!whole) {
                // of the CTAs that share the segment the last one folds what they left
                const int first_cta = owner(p.start), count = owner(p.start + p.pages - 1) - first_cta + 1;
                __threadfence();
                __syncwarp();
                if (lane == 0 && atomicAdd(static_cast<unsigned int*>(a.scratch) + first_cta, 1u) == (unsigned int)(count - 1)) folds[which] = first;
            }
        }
    }
    __syncthreads();
    const int folding = (folds[0] >= 0 ? 1 : 0) + (folds[1] >= 0 ? 1 : 0);
    if (folding == 0) {
        pdl_trigger();
        return;
    }
    __threadfence();
    // all warps for one segment, half of them each for two: of each 32 times 8 dims several warps share the pieces where there are more
    const int warps_here = kRowWarps / folding, own_warp = warp % warps_here, which = folding == 2 ? warp / warps_here : (folds[0] >= 0 ? 0 : 1);
    const Piece p = held[folds[which]];
    const int chunks = chunks_of(p), shares = max(1, warps_here / chunks), share = own_warp / chunks;
    float* const shared_by = parts + (size_t)(folding == 2 ? which * warps_here : 0) * kPiece;
    if (share < shares) {
        const int first_cta = owner(p.start), count = owner(p.start + p.pages - 1) - first_cta + 1;
        for (int chunk = own_warp % chunks; chunk < chunks; chunk += warps_here) {
            const int x = chunk * kWarp + lane, column = x / (HD / 8), d = x % (HD / 8) * 8;
            if (column >= p.columns) continue;
            Merged v;
            constexpr int kAtOnce = 4;
            for (int n0 = share; n0 < count; n0 += kAtOnce * shares) {
                float2 stats[kAtOnce];
                float4 lo[kAtOnce], hi[kAtOnce];
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) {
                    const int n = n0 + i * shares;
                    // (the segment begins in the first CTA's range, whose second piece it is)
                    const float* const from = left_by(first_cta + min(n, count - 1), n == 0 ? 1 : 0) + column * kPitch;
                    stats[i] = __ldcg(reinterpret_cast<const float2*>(from + HD));
                    lo[i] = __ldcg(reinterpret_cast<const float4*>(from + d));
                    hi[i] = __ldcg(reinterpret_cast<const float4*>(from + d + 4));
                }
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) {
                    if (n0 + i * shares < count) v.add(stats[i], lo[i], hi[i]);
                }
            }
            if (shares == 1) finish(p, column, d, v);
            else put(shared_by + (size_t)share * kPiece, column, d, v);
        }
    }
    __syncthreads();
    if (shares > 1) {
        for (int x = own_warp * kWarp + lane; x < p.columns * (HD / 8); x += warps_here * kWarp) {
            const int column = x / (HD / 8), d = x % (HD / 8) * 8;
            Merged v;
            for (int n = 0; n < shares; ++n) {
                const float* const from = shared_by + (size_t)n * kPiece + column * kPitch;
                v.add(*reinterpret_cast<const float2*>(from + HD), *reinterpret_cast<const float4*>(from + d), *reinterpret_cast<const float4*>(from + d + 4));
            }
            finish(p, column, d, v);
        }
    }
    pdl_trigger();
}

// Segments that a CTA each, or a cluster of 2, 4 or 8, gets through sooner than the ranges above get started: its warps share the
// segment's pages.  What the CTAs of a cluster leave is merged through distributed shared memory: no sums over the batch, no tickets, no
// way through the L2 and back.
template <int HD, bool E4M3>
__global__ void __launch_bounds__(kRowThreads, 2) kv8_few_rows_kernel(const Kv8AttentionArgs a, int blocks, int cluster) {
    using W = Walk<HD, E4M3, 1>;
    constexpr int kItems = HD / 8;                                                          // of a column
    extern __shared__ __align__(16) unsigned char smem[];
    float* const parts = reinterpret_cast<float*>(smem);                                    // a piece a warp, then the CTA's
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid / kWarp, 0);
    const int heads = a.cache.heads, group = a.query_heads / heads;
    const int number = (int)blockIdx.x / cluster, rank = (int)blockIdx.x - number * cluster, block = number % blocks;
    const int kv_head = number / blocks % heads, row = number / blocks / heads;
    pdl_wait();
    pdl_trigger();
    const RowWork w = row_work(a, row, group, W::kColumns);
    if (w.span.cut && tid == 0 && rank == 0 && block == 0 && kv_head == 0) atomicAdd(&g_kv8_range_errors, 1u);
    if (block >= w.blocks) return;                                                          // the whole cluster
    const Segment of{row, kv_head, block * W::kColumns, min(W::kColumns, w.span.count * group - block * W::kColumns), kv_head == 0 && block == 0};
    const int which = rank * kRowWarps + warp, warps = cluster * kRowWarps;
    const int page_first = (int)((long long)w.pages * which / warps), page_end = (int)((long long)w.pages * (which + 1) / warps);
    {
        W walk;
        if (page_first < page_end) walk.template run<false>(a, w, of, page_first, page_end);
        walk.keep(parts + (size_t)warp * W::kPiece, of.columns);
    }
    __syncthreads();
    auto finish = [&](Merged& v, int column, int d) {
        const float inverse = v.total == 0.0f ? 0.0f : 1.0f / v.total;
#pragma unroll
        for (int e = 0; e < 8; ++e) v.sum[e] *= inverse;
        write8<HD>(a, w.span.first, kv_head, of.column + column, d, v.sum);
    };
    float* const own = parts + (size_t)kRowWarps * W::kPiece;
    for (int x = tid; x < of.columns * kItems; x += kRowThreads) {
        const int column = x / kItems, d = x % kItems * 8;
        Merged v;
#pragma unroll
        for (int n = 0; n < kRowWarps; ++n) {
            const float* const from = parts + (size_t)n * W::kPiece + column * W::kPitch;
            v.add(*reinterpret_cast<const float2*>(from + HD), *reinterpret_cast<const float4*>(from + d), *reinterpret_cast<const float4*>(from + d + 4));
        }
        if (cluster == 1) {
            finish(v, column, d);
            continue;
        }
        float* const to = own + column * W::kPitch;
        *reinterpret_cast<float4*>(to + d) = make_float4(v.sum[0], v.sum[1], v.sum[2], v.sum[3]);
        *reinterpret_cast<float4*>(to + d + 4) = make_float4(v.sum[4], v.sum[5], v.sum[6], v.sum[7]);
        if (d == 0) *reinterpret_cast<float2*>(to + HD) = make_float2(v.top, v.total);
    }
    if (cluster == 1) return;
    tc::cluster_sync();
    for (int x = tid * cluster + rank; x < of.columns * kItems; x += kRowThreads * cluster) {
        const int column = x / kItems, d = x % kItems * 8;
        Merged v;
#pragma unroll 8
        for (int n = 0; n < cluster; ++n) {
            const uint32_t from = tc::peer_smem(tc::smem_u32(own + column * W::kPitch), (uint32_t)n);
            v.add(peer_float2(from + HD * 4), peer_float4(from + d * 4), peer_float4(from + d * 4 + 16));
        }
        finish(v, column, d);
    }
    tc::cluster_sync();                                                                     // no CTA leaves while another reads its memory
}

template <int HD, bool E4M3>
cudaError_t launch_few_rows(const Kv8AttentionArgs& a, int blocks, int cluster, cudaStream_t stream) {
    static std::atomic<unsigned long long> allowed{0};
    constexpr int kBytes = (kRowWarps + 1) * Walk<HD, E4M3, 1>::kPiece * (int)sizeof(float);
    const cudaError_t e = kv8_allow_smem(allowed, kv8_few_rows_kernel<HD, E4M3>, kBytes);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(blocks * a.cache.heads * a.rows * cluster));
    cfg.blockDim = dim3(kRowThreads);
    cfg.dynamicSmemBytes = kBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kv8_few_rows_kernel<HD, E4M3>, a, blocks, cluster);
}

template <int HD, bool E4M3, int TILES>
cudaError_t launch_rows(const Kv8AttentionArgs& a, cudaStream_t stream) {
    static std::atomic<unsigned long long> allowed{0};
    cudaError_t e = kv8_allow_smem(allowed, kv8_rows_kernel<HD, E4M3, TILES>, (int)rows_smem<HD, TILES>(Q3T_MAX_TABLE_ROWS));
    if (e == cudaSuccess) e = launch_pdl(kv8_zero_tickets_kernel, dim3(1), dim3(kRowCtas), 0, stream, static_cast<unsigned int*>(a.scratch));
    if (e != cudaSuccess) return e;
    e = launch_pdl(kv8_rows_kernel<HD, E4M3, TILES>, dim3(148 * rows_residency<HD, TILES>()), dim3(kRowThreads), rows_smem<HD, TILES>(a.rows), stream, a);
    return e != cudaSuccess || !a.prompts ? e : launch_kv8_prompts(a, HD, E4M3, stream);
}

// Which kernels a launch takes
struct Plan {
    int cluster;       // of kv8_few_rows_kernel; 0: not that one
    int blocks;        // its blocks of columns
    int tiles;         // of kv8_rows_kernel; 0: not that one either, the one row is a prompt
};
Plan plan_of(Kv8AttentionArgs& a, int head_dim) {
    const long long columns = (long long)a.most * (a.query_heads / a.cache.heads), blocks = (columns + kTileColumns - 1) / kTileColumns;
    const long long segments = blocks * a.cache.heads * a.rows;
    int cluster = kClusterCtas;
    while (cluster > 1 && (segments * cluster > kFewCtas || a.max_sequence <= kFewest * cluster)) cluster /= 2;
    a.prompts = 0;
    a.row_columns = INT_MAX;
    a.scratch_taken = kCounterBytes + kRowCtas * 2 * 2 * kTileColumns * (head_dim + 4) * (int)sizeof(float);
    if ((segments * cluster <= kFewCtas && a.max_sequence <= kFewTokens * cluster) || (segments <= (a.rows == 1 ? kOnePromptCtas : 2 * kFewCtas) && a.max_sequence <= kFewTokens / 2)) {
        return Plan{cluster, (int)blocks, 0};
    }
    if (columns > kRowColumns && ((long long)a.tokens * a.query_heads * a.max_sequence >= kPromptWork || a.max_sequence <= kShort)) {
        a.prompts = 1;
        a.row_columns = a.rows > 1 ? kRowColumns : 0;
        if (a.rows == 1) return Plan{0, 0, 0};
    }
    // Two tiles of columns a warp where rows may have more than one: what a page costs to read and to convert is paid once (one tile / two,
    // 64 rows of 2,048 tokens: 10 columns 94 / 73 us, 32 145 / 127; 16 rows of 512: 16 columns 20 / 21).  Beside prompts the others are mostly
    // single tokens, which fill one (63 of them and a prompt of 512: 44 / 52; 32 drafts of five and a prompt of 300: 38 / 35).
    return Plan{0, 0, !a.prompts && columns > kTileColumns ? 2 : 1};
}

template <int HD, bool E4M3>
cudaError_t launch_attention(const Kv8AttentionArgs& a, const Plan& plan, cudaStream_t stream) {
    if (plan.cluster > 0) return launch_few_rows<HD, E4M3>(a, plan.blocks, plan.cluster, stream);
    if (plan.tiles == 0) return launch_kv8_prompts(a, HD, E4M3, stream);
    return plan.tiles == 2 ? launch_rows<HD, E4M3, 2>(a, stream) : launch_rows<HD, E4M3, 1>(a, stream);
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
unsigned int kv8_prompt_page_error_count();
unsigned int kv8_prompt_range_error_count();
unsigned int kv8_range_error_count() {
    unsigned int v = 0;
    return cudaMemcpyFromSymbol(&v, g_kv8_range_errors, sizeof(v)) == cudaSuccess ? sum_of_counts({v, kv8_prompt_range_error_count()}) : ~0u;
}

}  // namespace q3t

extern "C" uint32_t q3t_kv8_page_error_count(void) {
    using namespace q3t;
    unsigned int v = 0;
    return cudaMemcpyFromSymbol(&v, g_kv8_page_errors, sizeof(v)) == cudaSuccess
               ? sum_of_counts({v, kv8_append_page_error_count(), kv8_prompt_page_error_count()}) : ~0u;
}

extern "C" size_t q3t_kv8_attention_scratch_bytes(const Q3tKv8AttentionDesc* desc) {
    q3t::Kv8AttentionArgs a;
    if (!q3t::attention_args(desc, &a)) return 0;
    q3t::plan_of(a, desc->cache->head_dimension);
    return a.scratch_taken + (a.prompts ? q3t::kv8_prompt_scratch_bytes(a.max_sequence, desc->cache->head_dimension) : 0);
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
    const Plan plan = plan_of(a, desc->cache->head_dimension);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool e4m3 = desc->cache->format == Q3T_KV8_E4M3;
    if (desc->cache->head_dimension == 128) {
        return static_cast<int32_t>(e4m3 ? launch_attention<128, true>(a, plan, s) : launch_attention<128, false>(a, plan, s));
    }
    return static_cast<int32_t>(e4m3 ? launch_attention<64, true>(a, plan, s) : launch_attention<64, false>(a, plan, s));
}
