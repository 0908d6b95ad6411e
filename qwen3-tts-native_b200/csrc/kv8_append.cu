// Keys and values of new tokens, quantised into the pages of an 8-bit cache (q3t_launch_kv8_append).
//
// One warp quantises what a launch adds to one page in one head of one plane: its new tokens (up to 16 x head_dim bf16) are read once
// and stay in registers from the largest magnitude to the codes, so the traffic is the floor's, two bytes in and one out.
//   scale = max(amax / M, 2^-126); code = round(x * (1 / scale)); with tokens held in the page's lower slots the scale is the
//   larger of that and the page's own, and where it has grown the held codes are rounded again.
// The reciprocal is taken once a page and head: a division a value would cost more issue slots than the memory takes time.  2^-126
// keeps it finite and makes a page of zeros no special case.
// The page's first new token (its slot's page is not the token's before) owns the page; a warp looks for owners in a window of
// consecutive tokens and takes them one after the other.  Where every token owns a page (a decode step) small windows let the pages'
// chains of loads run side by side; where one or two of 16 do (a prompt) large ones spare warps that find nothing.  The host does not
// know which it is, only how many warps windows of one token would take (tokens x 2 x heads), so the window grows where that many no
// longer run at once: 4 from 2^14 on and 16 from 2^16 on.  Measured with 8 heads of 128, int8, in us, windows of 1 / 4 / 16:
//   a prompt of 512 tokens 4.5 / 4.1 / 4.5, of 1,024 6.2 / 4.6 / 4.5, of 2,048 9.2 / 5.7 / 4.8, of 4,096 15.4 / 8.4 / 5.8, of 8,192 27.8 / 13.7 / 8.8;
//   512 rows of one token 8.0 / 8.7 / 21, 1,024 14.1 / 14.0 / 21, 2,048 26.0 / 23.0 / 28, 4,096 51.8 / 43.9 / 50.3.
//
// What bounds it: a decode step the latency of five loads and sums one behind the other (64 rows: 3.0 us); a large batch memory (49,174
// tokens in 43 rows, 303 MB: 54.5 us, 5.6 TB/s, on inputs that change from call to call 58; three CTAs an SM instead of four, with more
// registers, take 12 % longer).  A prompt of 1,500 tokens takes 4.8 us (4 an SM: 5.1).

#include "kv8.cuh"
#include "q3t_kernels.cuh"

namespace q3t {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kAppendWarps = kAppendThreads / kWarp;
constexpr long long kManyWarps = 1 << 14, kMostWarps = 1 << 16;      // windows of 4 and of 16 tokens from here on

__device__ unsigned int g_kv8_nonfinite = 0;
__device__ unsigned int g_kv8_append_page_errors = 0;

struct AppendArgs {
    Kv8View cache;
    const bf16* key;
    const bf16* value;
    const long long* slots;
    const int* token_count;
    int tokens;
    int key_stride, value_stride;
};

// 16 bytes that are read once; not by the read-only path, since a launch ahead of this one may have written them
__device__ __forceinline__ int4 load_once(const void* p) {
    int4 v;
    asm volatile("ld.global.L1::no_allocate.v4.s32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}

// int8 of four values of magnitude 127 and less: adding 1.5 * 2^23 rounds to nearest even and leaves the integer in the low byte
__device__ __forceinline__ uint32_t pack_int8(float a, float b, float c, float d) {
    const float magic = 12582912.0f;
    const uint32_t ab = __byte_perm(__float_as_uint(__fadd_rn(a, magic)), __float_as_uint(__fadd_rn(b, magic)), 0x0040);
    const uint32_t cd = __byte_perm(__float_as_uint(__fadd_rn(c, magic)), __float_as_uint(__fadd_rn(d, magic)), 0x0040);
    return __byte_perm(ab, cd, 0x5410);
}
template <bool E4M3>
__device__ __forceinline__ uint32_t pack_codes(float a, float b, float c, float d) {
    if (E4M3) return to_e4m3x2(a, b) | (to_e4m3x2(c, d) << 16);
    return pack_int8(a, b, c, d);
}
// four codes as fp32
template <bool E4M3>
__device__ __forceinline__ void unpack_codes(uint32_t word, float (&v)[4]) {
    if (E4M3) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t pair = e4m3_to_half2(word >> (16 * i));
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&pair));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = static_cast<float>(static_cast<signed char>(word >> (8 * i)));
    }
}

template <int HD, bool E4M3, int WINDOW>
__global__ void __launch_bounds__(kAppendThreads, WINDOW == 4 ? 3 : 4) kv8_append_kernel(const AppendArgs a) {
    constexpr int kLanes = HD / 8;                        // of a token: 8 values each
    constexpr int kAtOnce = kWarp / kLanes;               // tokens
    constexpr int kRounds = kPageTokens / kAtOnce;
    constexpr float kMost = E4M3 ? 448.0f : 127.0f;
    __shared__ int newest[kAppendWarps][kPageTokens];     // of each slot of the page: the token that fills it, or -1
    const int lane = threadIdx.x % kWarp, warp = threadIdx.x / kWarp;
    pdl_wait();
    pdl_trigger();
    const int count = a.token_count != nullptr ? min(max(*a.token_count, 0), a.tokens) : a.tokens;
    const long long item = (long long)blockIdx.x * kAppendWarps + warp;
    const int heads = a.cache.heads;
    const long long window = item / (2 * heads);
    const int rest = (int)(item - window * 2 * heads);
    const bool values = rest >= heads;
    const int head = values ? rest - heads : rest;
    if (window * WINDOW >= count) return;
    const int t0 = (int)window * WINDOW;
    // the page of a token's slot, or -1
    auto page_at = [&](int t, int& slot) {
        const long long s = t >= 0 && t < count ? a.slots[t] : -1;
        slot = (int)(s & (kPageTokens - 1));
        const long long page = s >> 4;
        return s < 0 ? -1 : page < a.cache.pages ? (int)page : -2;
    };
    static_assert(kPageTokens == 16, "page_at");
    int slot;
    const int page_here = lane <= WINDOW ? page_at(t0 - 1 + lane, slot) : -1;
    const unsigned int bad = __ballot_sync(0xffffffffu, lane > 0 && page_here == -2);
    if (rest == 0 && bad != 0u && lane == 0) atomicAdd(&g_kv8_append_page_errors, (unsigned int)__popc(bad));
    const int page_before = __shfl_up_sync(0xffffffffu, page_here, 1);
    unsigned int owners = __ballot_sync(0xffffffffu, lane > 0 && page_here >= 0 && page_here != page_before);

    while (owners != 0u) {
        const int which = __ffs(owners) - 1;
        owners &= owners - 1;
        const int page = __shfl_sync(0xffffffffu, page_here, which);
        // ---- which token fills which slot: of the tokens that stand together the last one that names it
        if (lane < kPageTokens) newest[warp][lane] = -1;
        __syncwarp();
        for (int base = t0 - 1 + which;;) {
            const bool same = page_at(base + lane, slot) == page;
            const unsigned int apart = __ballot_sync(0xffffffffu, !same);
            const int run = apart != 0u ? __ffs(apart) - 1 : kWarp;
            const unsigned int peers = __match_any_sync(0xffffffffu, lane < run ? slot : kWarp + lane);
            if (lane < run && (peers >> lane) == 1u) newest[warp][slot] = base + lane;
            __syncwarp();
            if (run < kWarp) break;
            base += kWarp;
        }
        const int mine = lane < kPageTokens ? newest[warp][lane] : -1;
        const int held = __ffs(__ballot_sync(0xffffffffu, mine >= 0)) - 1;       // slots below the new tokens
        __syncwarp();
        const bf16* source = (values ? a.value : a.key) + (size_t)head * HD + (lane % kLanes) * 8;
        const size_t stride = values ? a.value_stride : a.key_stride;
        uint8_t* const codes = (values ? a.cache.v : a.cache.k) + (long long)page * a.cache.page_stride + (size_t)head * (kPageTokens * HD)
                               + (lane / kLanes) * HD + (lane % kLanes) * 8;
        float* const scale_at = (values ? a.cache.v_scales : a.cache.k_scales) + (long long)page * a.cache.scale_stride + head;
        const float own = held > 0 ? *scale_at : 0.0f;
        uint32_t x[kRounds][4];
        bool filled[kRounds];
#pragma unroll
        for (int i = 0; i < kRounds; ++i) {
            const int t = __shfl_sync(0xffffffffu, mine, i * kAtOnce + lane / kLanes);
            filled[i] = t >= 0;
            int4 v = make_int4(0, 0, 0, 0);
            if (t >= 0) v = load_once(source + (size_t)t * stride);
            x[i][0] = (uint32_t)v.x;
            x[i][1] = (uint32_t)v.y;
            x[i][2] = (uint32_t)v.z;
            x[i][3] = (uint32_t)v.w;
        }
        // ---- the largest magnitude: bf16 without its sign compares like an integer
        auto largest = [&]() {
            uint32_t most = 0u;
#pragma unroll
            for (int i = 0; i < kRounds; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) most = __vmaxu2(most, x[i][j] & 0x7fff7fffu);
            }
            return __reduce_max_sync(0xffffffffu, max(most & 0xffffu, most >> 16));
        };
        unsigned int most = largest();
        if (most >= 0x7f80u) {                            // infinities and NaN among them
            if (lane == 0) atomicAdd(&g_kv8_nonfinite, 1u);
#pragma unroll
            for (int i = 0; i < kRounds; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) x[i][j] = __vminu2(x[i][j] & 0x7fff7fffu, 0x7f7f7f7fu) | (x[i][j] & 0x80008000u);
            }
            most = largest();
        }
        const float fresh = fmaxf(__fdiv_rn(__uint_as_float(most << 16), kMost), kKv8SmallestScale);
        const float scale = held > 0 ? fmaxf(own, fresh) : fresh;
        const float inverse = __frcp_rn(scale);
        if (held > 0 && scale > own) {
            const float shrink = __fmul_rn(own, inverse);
#pragma unroll
            for (int i = 0; i < kRounds; ++i) {
                if (i * kAtOnce + lane / kLanes < held) {
                    uint2* const at = reinterpret_cast<uint2*>(codes + i * kAtOnce * HD);
                    uint2 w = *at;
                    float f[4];
                    unpack_codes<E4M3>(w.x, f);
                    w.x = pack_codes<E4M3>(__fmul_rn(f[0], shrink), __fmul_rn(f[1], shrink), __fmul_rn(f[2], shrink), __fmul_rn(f[3], shrink));
                    unpack_codes<E4M3>(w.y, f);
                    w.y = pack_codes<E4M3>(__fmul_rn(f[0], shrink), __fmul_rn(f[1], shrink), __fmul_rn(f[2], shrink), __fmul_rn(f[3], shrink));
                    *at = w;
                }
            }
        }
        if (lane == 0 && (held == 0 || scale > own)) *scale_at = scale;
#pragma unroll
        for (int i = 0; i < kRounds; ++i) {
            uint2 w;
            w.x = pack_codes<E4M3>(__fmul_rn(bf_lo(x[i][0]), inverse), __fmul_rn(bf_hi(x[i][0]), inverse),
                                   __fmul_rn(bf_lo(x[i][1]), inverse), __fmul_rn(bf_hi(x[i][1]), inverse));
            w.y = pack_codes<E4M3>(__fmul_rn(bf_lo(x[i][2]), inverse), __fmul_rn(bf_hi(x[i][2]), inverse),
                                   __fmul_rn(bf_lo(x[i][3]), inverse), __fmul_rn(bf_hi(x[i][3]), inverse));
            if (filled[i]) *reinterpret_cast<uint2*>(codes + i * kAtOnce * HD) = w;
        }
    }
}

template <int HD, bool E4M3>
cudaError_t launch_append(const AppendArgs& a, cudaStream_t stream) {
    const long long heads = 2 * a.cache.heads, most = heads * a.tokens;
    const int window = most < kManyWarps ? 1 : most < kMostWarps ? 4 : kPageTokens;
    const long long warps = (a.tokens + window - 1) / window * heads;
    const dim3 grid((unsigned)((warps + kAppendWarps - 1) / kAppendWarps)), block(kAppendThreads);
    return window == 1 ? launch_pdl(kv8_append_kernel<HD, E4M3, 1>, grid, block, 0, stream, a)
           : window == 4 ? launch_pdl(kv8_append_kernel<HD, E4M3, 4>, grid, block, 0, stream, a)
                         : launch_pdl(kv8_append_kernel<HD, E4M3, kPageTokens>, grid, block, 0, stream, a);
}

}  // namespace

unsigned int kv8_append_page_error_count() {
    unsigned int v = 0;
    return cudaMemcpyFromSymbol(&v, g_kv8_append_page_errors, sizeof(v)) == cudaSuccess ? v : ~0u;
}

}  // namespace q3t

extern "C" uint32_t q3t_kv8_nonfinite_count(void) {
    unsigned int v = 0;
    return cudaMemcpyFromSymbol(&v, q3t::g_kv8_nonfinite, sizeof(v)) == cudaSuccess ? v : ~0u;
}

extern "C" int32_t q3t_launch_kv8_append(const Q3tKv8Cache* cache, const uint16_t* key, const uint16_t* value, const int64_t* slots,
                                         const int32_t* token_count, int32_t tokens, int32_t key_stride, int32_t value_stride,
                                         void* stream) {
    using namespace q3t;
    AppendArgs a;
    if (!kv8_view(cache, &a.cache) || key == nullptr || value == nullptr || slots == nullptr || tokens < 1) return cudaErrorInvalidValue;
    const int width = cache->key_value_heads * cache->head_dimension;
    a.key = reinterpret_cast<const bf16*>(key);
    a.value = reinterpret_cast<const bf16*>(value);
    a.slots = reinterpret_cast<const long long*>(slots);
    a.token_count = token_count;
    a.tokens = tokens;
    a.key_stride = key_stride != 0 ? key_stride : width;
    a.value_stride = value_stride != 0 ? value_stride : width;
    if (a.key_stride < width || a.value_stride < width || a.key_stride % 8 != 0 || a.value_stride % 8 != 0
        || (reinterpret_cast<uintptr_t>(key) | reinterpret_cast<uintptr_t>(value)) % 16 != 0 || reinterpret_cast<uintptr_t>(slots) % 8 != 0
        || (long long)tokens * 2 * cache->key_value_heads > (1ll << 33)) {
        return cudaErrorInvalidValue;
    }
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool e4m3 = cache->format == Q3T_KV8_E4M3;
    if (cache->head_dimension == 128) return static_cast<int32_t>(e4m3 ? launch_append<128, true>(a, s) : launch_append<128, false>(a, s));
    return static_cast<int32_t>(e4m3 ? launch_append<64, true>(a, s) : launch_append<64, false>(a, s));
}
