// Causal attention over an 8-bit paged cache (q3t_launch_kv8_attention): rows of many new tokens.  The formula, and what makes a page's
// value scale an addend of the exponent, are in kv8_attention.cu.
//
// A CTA takes 256 columns ((new token, query head) pairs of a KV head, two tiles of 128 rows of the tensor cores) of a row and walks
// what they see of its cache once, 128 tokens a step, two halves of 64:
//   copies    codes from their pages to registers, to fp16 (exact) and into shared memory, swizzled: K by four warps, V by four; the
//             next step's are requested before the present one's are stored
//   scores    S = Q K^T, tcgen05.mma from shared memory into 64 columns of tensor memory a tile and half
//   softmax   a thread a row: w = exp2(s * key scale + log2(value scale) - reference) as fp16 over the scores' place
//   output    O += W V, the weights from tensor memory
// While a tile's half is in the softmax the products of its other half and of the other tile run.  A row's reference follows its scores
// only when its weights outgrow fp16, so that the output in tensor memory is rescaled almost never.
//
// Where the blocks of 256 columns are fewer than the SMs they become blocks of 128, and where each could have several SMs to itself and rows may see
// 2,048 tokens and more, their steps are cut into parts, which kv8_join_kernel merges.
//
// What bounds it: of a half's 2,000 cycles (1,550 with one tile, heads of 128) the tensor cores take 1,024 and the exponentials as much, on units that
// run side by side.  Shared memory is a third: at 128 bytes a cycle a score product of 64 tokens has its operands, 6 KB, in 48 cycles and is
// done in 32, which makes the products 1,280, and the copies' stores are 256 more (arithmetic, not measured apart).  The rest is
// the way of a tile's half through barriers, tensor memory and registers, of which two tiles hide one in the other
// what two can.  A block costs 7 us more before and after its steps.  A chunk of 4,096 tokens over 16,384 (16 query heads, 8 KV heads of 128): 472 us,
// 1,018 TFLOP/s (call after call for long enough that the power limit shows: 517 us, 930); 11 prompts of 667 to 1,333 over 1,400 to 3,333 (32, 8): 415 us;
// a prompt of 1,500: 27.5 us; 256 tokens over 16,384: 51 us.

#include "kv8.cuh"
#include "q3t_kernels.cuh"
#include "q3t_tcgen05.cuh"

namespace q3t {
namespace {

constexpr int kTileRows = 128;
constexpr int kStep = 128;                              // tokens
constexpr int kStepPages = kStep / kPageTokens;
constexpr int kHalf = kStep / 2, kHalfPages = kStepPages / 2;
constexpr int kPromptThreads = 640;                     // warps 0..7 softmax (a tile each four), 8..11 K, 12..15 V, 16 and 17 products (a tile each)
constexpr int kSoftmaxWarps = 8, kKeyWarp = 8, kValueWarp = 12, kProductWarp = 16;
// What setmaxnreg hands out is what the block was launched with
constexpr int kLaunchRegisters = 96, kSoftmaxRegisters = 144, kCopyRegisters = 72, kProductRegisters = 48;
static_assert(2 * kSoftmaxRegisters + 2 * kCopyRegisters + kProductRegisters <= 5 * kLaunchRegisters, "registers of the five warpgroups");
constexpr int kScaleRing = 4;                           // steps whose scales are kept: K runs two steps ahead of the softmax
constexpr uint32_t kTmemCols = 512, kOut = 256;         // scores of the tiles at 0 and 128, outputs at 256 and 384
// A launch has as many parts as its longest row may have of so many tokens, and a row takes as many of them as it has steps.  (Bound of 16,384, 256
// tokens, parts of 1, 2, 4 and 8 steps and more in us: over 300 16.8 / 17.8 / 17.7 / 17.7, over 1,024 20.1 / 21.7 / 28.6 / 28.5, over 2,000 23.1 / 25.0 / 26.4 / 45.6.)
constexpr int kPartTokens = 1024;
constexpr float kMostWeight = 32768.0f;                 // of a page's weights together
constexpr long long kBudgetCycles = 4000000000ll;        // about two seconds

std::atomic<int> g_lost_block{-1};
__device__ unsigned int g_kv8_prompt_errors = 0;
__device__ unsigned int g_kv8_prompt_page_errors = 0;
__device__ unsigned int g_kv8_prompt_range_errors = 0;

template <int HD>
struct PromptSmem {
    static constexpr int kQueryBytes = 2 * kTileRows * HD * 2;
    static constexpr int kTileBytes = kStep * HD * 2;
    static constexpr size_t kBytes = 1024 + kQueryBytes + 4 * kTileBytes;
};

// As tc::Guard, but the clock is looked at whenever a look at a barrier ends: one of a whole warp may be suspended for milliseconds, a
// thousand of which are no bound.  (With a limit to the suspension, 20 us, a chunk of 4096 at 16k took 6 % longer.)
struct Guard {
    long long deadline;                                                // of clock64()
    volatile int* abort_flag;
    __device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity) const {
        while (!tc::mbar_try_wait(bar, parity)) {
            if (*abort_flag != 0) return false;
            if (clock64() > deadline) {
                *abort_flag = 1;
                return false;
            }
        }
        return true;
    }
};

struct Item {
    int row, kv_head, block, part;
    RowSpan span;
};

// How a launch is cut: blocks of 128 or 256 columns, and what they see into so many parts at most
struct PromptCut {
    int block_columns, parts;
    long long items;
};

// What an item's parts leave is 16 bytes of each row for 4 dims at a time, then the rows' references and sums; kv8_join_kernel learns from
// the first part what there is to join
struct Joint {
    int parts;         // fewer than two: nothing
    int columns, column0;
    int kv_head, first;
    int unused[3];
};
constexpr int kMostParts = 8;
constexpr int kJointBytes = 148 * (int)sizeof(Joint);
template <int HD>
struct Part {
    static constexpr size_t kFloats = (size_t)2 * kTileRows * (HD + 2);
};

// 16-byte piece `piece` of row `t` of a tile of 128: 64 dims in 128 bytes, swizzled, the next 64 a tile of rows further on
__device__ __forceinline__ uint32_t tile_offset(int t, int piece) {
    return (uint32_t)((piece >> 3) * kTileRows * 128 + t * 128 + (((piece & 7) ^ (t & 7)) << 4));
}
static_assert(kStep == kTileRows, "tile_offset");
// B operand whose rows (dims) are contiguous: 64 of them in 128 bytes, the next 64 a tile of tokens further on, eight of K 1024 bytes
__device__ __forceinline__ uint64_t desc_rows_contiguous(uint32_t smem) {
    return (uint64_t)((smem >> 4) & 0x3FFFu) | ((uint64_t)(kStep * 128 / 16) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// 16 or 32 columns of this thread's lane, to be waited for
__device__ __forceinline__ void tmem_load_16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_load_32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
          "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
template <int N>
__device__ __forceinline__ void tmem_wait_load(uint32_t (&r)[N]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));        // not to be used ahead of the wait
}
__device__ __forceinline__ void tmem_store_8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_store_16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// PARTS: items may come in parts (without: two divisions and a branch an item fewer, 1.3 us of a prompt of 1,500 tokens).  lost_block: the one that
// ends as if a wait of its had run out, -1: none
template <int HD, bool E4M3, bool PARTS>
__global__ void __launch_bounds__(kPromptThreads, 1) kv8_prompt_kernel(const Kv8AttentionArgs a, const int block_columns, const int parts_asked, unsigned char* const left,
                                                                       const int lost_block) {
    const int most_parts = PARTS ? parts_asked : 1;
    using Smem = PromptSmem<HD>;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* const smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    unsigned char* const queries = smem;                               // [tile]
    unsigned char* const keys = smem + Smem::kQueryBytes;              // [step % 2]
    unsigned char* const values = keys + 2 * Smem::kTileBytes;         // [step % 2]
    __shared__ float4 scales[kScaleRing][kStepPages];                  // of each page: key scale, log2 and reciprocal of the value scale, what its weights miss
    // full: V of a step and K of the next one
    __shared__ uint64_t first_k, full[2], empty_k[2], empty_v[2], s_ready[2][2], p_ready[2][2], o_ready[2][2], q_ready;     // [tile][half]
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    __shared__ int warp_items[kPromptThreads / kWarp];
    __shared__ Item found;
    volatile int* const abort_flag = &abort_word;

    const int tid = threadIdx.x, lane = tid % kWarp, warp = __shfl_sync(0xffffffffu, tid / kWarp, 0);
    const int heads = a.cache.heads, group = a.query_heads / heads;

    // ---- this CTA's columns: the rows of many columns have ceil(columns / block_columns) items a KV head; those of a row's last tokens, which see
    // the most, first, all KV heads of a block together
    if (a.row_columns == 0) pdl_wait();                                // (else the launch ahead has waited and counts what lies outside the host's bounds)
    if (tid == 0) found.row = -1;
    __syncthreads();
    int sum = 0;
    for (int first = 0; first < a.rows; first += kPromptThreads) {
        const int row = first + tid;
        int mine = 0, own = 0;
        RowSpan span{};
        if (row < a.rows) {
            span = row_span(a.starts, a.lengths, row, a.tokens, a.most, a.max_sequence);
            const long long columns = (long long)span.count * group;
            if (a.row_columns == 0 && span.cut && blockIdx.x == 0) atomicAdd(&g_kv8_prompt_range_errors, 1u);
            own = columns > a.row_columns ? (int)((columns + block_columns - 1) / block_columns) * heads * most_parts : 0;
            mine = own;
        }
#pragma unroll
        for (int o = 1; o < kWarp; o <<= 1) {
            const int other = __shfl_up_sync(0xffffffffu, mine, o);
            if (lane >= o) mine += other;
        }
        if (lane == kWarp - 1) warp_items[warp] = mine;
        __syncthreads();
        for (int w = 0; w < warp; ++w) mine += warp_items[w];
        const int to = sum + mine, from = to - own, at = (int)blockIdx.x;
        if (at >= from && at < to) {
            const int number = (at - from) / most_parts;
            found = Item{row, number % heads, own / most_parts / heads - 1 - number / heads, (at - from) % most_parts, span};
        }
        for (int w = 0; w < kPromptThreads / kWarp; ++w) sum += warp_items[w];
        __syncthreads();
    }
    const Item item = found;
    Joint* const joint = reinterpret_cast<Joint*>(left) + (int)blockIdx.x / most_parts;
    if (item.row < 0) {                                                // (a grid is as large as tokens and rows may need)
        if (most_parts > 1 && tid == 0 && (int)blockIdx.x % most_parts == 0) joint->parts = 0;
        pdl_wait();                                                    // what follows relies on this launch to be behind the one before
        return;
    }
    const int column0 = item.block * block_columns;
    const int columns = min(block_columns, item.span.count * group - column0);
    // of column r of the item the token, among the row's new ones, and the head among the KV head's: one division, and a product that is
    // exact for what is below 320
    const int token0 = column0 / group, rest0 = column0 - token0 * group;
    const float per_group = 1.0f / static_cast<float>(group);
    auto place_of = [&](int r, int& head) {
        const int more = (int)((static_cast<float>(rest0 + r) + 0.5f) * per_group);
        head = rest0 + r - more * group;
        return token0 + more;
    };
    auto seen_by = [&](int r) {
        int head;
        return min(max(item.span.base + place_of(r, head) + 1, 0), a.max_sequence);
    };
    // (both tiles go as far as the second one's last column sees; one that is empty not at all)
    const int tiles = columns > kTileRows ? 2 : 1;
    const int all_halves = (seen_by(columns - 1) + kHalf - 1) / kHalf, all_steps = (all_halves + 1) / 2, parts = PARTS ? max(1, min(most_parts, all_steps)) : 1;
    if (most_parts > 1 && tid == 0 && item.part == 0) *joint = Joint{parts, columns, column0, item.kv_head, item.span.first, {0, 0, 0}};
    if (item.part >= parts) {
        pdl_wait();
        return;
    }
    // this part's steps; what follows counts them from 0
    const int step0 = all_steps * item.part / parts, steps = all_steps * (item.part + 1) / parts - step0;
    const int halves = min(2 * steps, all_halves - 2 * step0);

    Guard guard;
    guard.deadline = clock64() + kBudgetCycles;
    guard.abort_flag = abort_flag;
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(&full[i], 8);
            tc::mbar_init(&empty_k[i], tiles);
            tc::mbar_init(&empty_v[i], tiles);
            for (int h = 0; h < 2; ++h) {
                tc::mbar_init(&s_ready[i][h], 1);
                tc::mbar_init(&p_ready[i][h], 4);
                tc::mbar_init(&o_ready[i][h], 1);
            }
        }
        tc::mbar_init(&first_k, 4);
        tc::mbar_init(&q_ready, kSoftmaxWarps);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kProductWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(&tmem_slot)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_slot;

    if (warp >= kKeyWarp && warp < kProductWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kCopyRegisters));
        // ---- copies: a thread takes 16 codes (8 of a head of 64) of one token of each of a step's pages.  Eight threads that store side by
        // side have half of the parts of two tokens, which the swizzle puts into all of the banks
        const bool is_value = warp >= kValueWarp;
        const int t = tid - (is_value ? kValueWarp : kKeyWarp) * kWarp;
        const int token = ((t >> 2) & 1) | ((t >> 4) << 1), part = (t & 3) | (((t >> 3) & 1) << 2);
        constexpr int kCodes = HD / 8;                                 // bytes a thread and token
        const int store_at = (int)tile_offset(token, kCodes == 16 ? 2 * part : part);
        const int store_more = (int)tile_offset(token, 2 * part + 1) - store_at;
        const uint8_t* const plane = (is_value ? a.cache.v : a.cache.k) + (size_t)item.kv_head * (kPageTokens * HD) + token * HD + part * kCodes;
        unsigned char* const buffers = is_value ? values : keys;
        uint64_t* const empty = is_value ? empty_v : empty_k;
        const int last = min(max(item.span.base + item.span.count, 0), a.max_sequence);        // what lies behind may read as NaN
        const int page0 = step0 * kStepPages;
        const bool last_block = column0 + block_columns >= item.span.count * group;
        const int* const ids_at = a.table + (size_t)item.row * a.table_stride;
        int ids = -1;                                                  // of 32 pages, a lane each
        int4 code[kStepPages];
        uint32_t good = 0u;                                            // pages of the step that are there
        auto request = [&](int step) {
            if (step % (kWarp / kStepPages) == 0) {
                const int page = page0 + step * kStepPages + lane;
                ids = page * kPageTokens < last ? ids_at[page] : -1;
                if (ids < 0 || ids >= a.cache.pages) {
                    if (page * kPageTokens < last && page < page0 + steps * kStepPages && t < kWarp && !is_value && item.kv_head == 0 && last_block) {
                        atomicAdd(&g_kv8_prompt_page_errors, 1u);
                    }
                    ids = -1;
                }
            }
            good = 0u;
#pragma unroll
            for (int p = 0; p < kStepPages; ++p) {
                const int id = __shfl_sync(0xffffffffu, ids, step % (kWarp / kStepPages) * kStepPages + p);
                code[p] = make_int4(0, 0, 0, 0);
                if (id >= 0 && (page0 + step * kStepPages + p) * kPageTokens + token < last) {
                    const uint8_t* const from = plane + (long long)id * a.cache.page_stride;
                    if (kCodes == 16) {
                        asm volatile("ld.global.L1::no_allocate.v4.s32 {%0,%1,%2,%3}, [%4];" : "=r"(code[p].x), "=r"(code[p].y), "=r"(code[p].z), "=r"(code[p].w) : "l"(from));
                    } else {
                        const int2 half = *reinterpret_cast<const int2*>(from);
                        code[p].x = half.x;
                        code[p].y = half.y;
                    }
                }
                good |= id >= 0 ? 1u << p : 0u;
            }
        };
        float key_scale = 0.0f, value_scale = 0.0f;
        // a page's scales, by one thread of the keys'
        auto request_scales = [&](int step) {
            const int id = __shfl_sync(0xffffffffu, ids, step % (kWarp / kStepPages) * kStepPages + (t & 7));
            if (t < kStepPages && !is_value && id >= 0) {
                const long long at = (long long)id * a.cache.scale_stride + item.kv_head;
                key_scale = a.cache.k_scales[at];
                value_scale = a.cache.v_scales[at];
            }
        };
        if (steps > 0) {
            request(0);
            request_scales(0);
        }
        for (int step = 0; step < steps; ++step) {
            const int buffer = step & 1;
            if (step >= 2 && !__all_sync(0xffffffffu, guard.wait(&empty[buffer], ((step >> 1) - 1) & 1))) break;
            if (t < kStepPages && !is_value) {
                // a page that is not there weighs nothing: its codes are zeros, its value scale is as well
                const float vs = fmaxf(value_scale, kKv8LeastValueScale), back = fminf(value_scale * (1.0f / kKv8LeastValueScale), 1.0f);
                scales[step % kScaleRing][t] = (good >> t) & 1u ? make_float4(key_scale, log2_fast(vs), reciprocal_fast(vs), back)
                                                               : make_float4(0.0f, -INFINITY, 0.0f, 1.0f);
            }
            unsigned char* const tile = buffers + buffer * Smem::kTileBytes + store_at;
#pragma unroll
            for (int p = 0; p < kStepPages; ++p) {
                uint32_t h[8];
                codes_to_half<E4M3>((uint32_t)code[p].x, h[0], h[1]);
                codes_to_half<E4M3>((uint32_t)code[p].y, h[2], h[3]);
                *reinterpret_cast<int4*>(tile + p * (kPageTokens * 128)) = make_int4((int)h[0], (int)h[1], (int)h[2], (int)h[3]);
                if (kCodes == 16) {
                    codes_to_half<E4M3>((uint32_t)code[p].z, h[4], h[5]);
                    codes_to_half<E4M3>((uint32_t)code[p].w, h[6], h[7]);
                    *reinterpret_cast<int4*>(tile + store_more + p * (kPageTokens * 128)) = make_int4((int)h[4], (int)h[5], (int)h[6], (int)h[7]);
                }
            }
            // (ahead of the next requests: the fence would wait for them)
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(is_value ? &full[buffer] : step == 0 ? &first_k : &full[buffer ^ 1]);
            if (step + 1 < steps) {
                request(step + 1);
                request_scales(step + 1);
            }
        }
        // the last step has no next K; its barrier's phase before is past when the scores of the step before last are there
        if (!is_value && steps > 0) {
            if (steps > 1) guard.wait(&empty_k[steps & 1], ((steps - 2) >> 1) & 1);
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&full[(steps - 1) & 1]);
        }
    } else if (warp >= kProductWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kProductRegisters));
        const int tile = warp - kProductWarp;
        if (tile < tiles && steps > 0 && tc::elect_one()) {
            // ---- products of a tile: both operands fp16, sums fp32.  What a step takes here is the looks at barriers, 350 cycles each beside the
            // copies' stores: hence a thread a tile (one for both took 30 % longer), and one barrier for V and the next K.
            const uint32_t scores_idesc = (1u << 4) | ((uint32_t)(kHalf >> 3) << 17) | ((uint32_t)(kTileRows >> 4) << 24);
            // B with its rows (dims) contiguous: bit 16
            const uint32_t out_idesc = (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(kTileRows >> 4) << 24);
            const uint32_t q = tc::smem_u32(queries) + tile * kTileRows * HD * 2;
            auto scores = [&](int n) {                                 // n: half of a step, counted through
                const uint32_t k = tc::smem_u32(keys) + ((n >> 1) & 1) * Smem::kTileBytes + (n & 1) * kHalf * 128;
#pragma unroll
                for (int j = 0; j < HD / 16; ++j) {
                    umma_ss(tmem + tile * kStep + (n & 1) * kHalf, tc::umma_desc(q + (j / 4) * kTileRows * 128 + 32 * (j % 4)),
                            tc::umma_desc(k + (j / 4) * kStep * 128 + 32 * (j % 4)), scores_idesc, j != 0 ? 1u : 0u);
                }
                tc::umma_commit(&s_ready[tile][n & 1]);
                if ((n & 1) != 0 || n + 1 == halves) tc::umma_commit(&empty_k[(n >> 1) & 1]);
            };
            bool ok = guard.wait(&q_ready, 0) && guard.wait(&first_k, 0);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (ok) {
                scores(0);
                if (halves > 1) scores(1);
            }
            for (int n = 0; n < halves && ok; ++n) {
                const int step = n >> 1, h = n & 1;
                ok = (h != 0 || guard.wait(&full[step & 1], (step >> 1) & 1)) && guard.wait(&p_ready[tile][h], step & 1);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t v = tc::smem_u32(values) + (step & 1) * Smem::kTileBytes + h * kHalf * 128;
#pragma unroll
                for (int j = 0; j < kHalf / 16; ++j) {
                    tc::umma_f16_ts(tmem + kOut + tile * 128, tmem + tile * kStep + h * kHalf + 8 * j, desc_rows_contiguous(v + j * 16 * 128), out_idesc,
                                    (n | j) != 0 ? 1u : 0u);
                }
                tc::umma_commit(&o_ready[tile][h]);
                if (h != 0 || n + 1 == halves) tc::umma_commit(&empty_v[step & 1]);
                if (n + 2 >= halves) continue;
                // the next scores of this half lie over the weights: products of other accumulators are in no order of their own
                ok = guard.wait(&o_ready[tile][h], step & 1);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (ok) scores(n + 2);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegisters));
        // ---- queries to fp16, by a power of two that brings the largest of each to 2^7..2^8
        constexpr int kLanes = HD / 8, kAtOnce = kWarp / kLanes;       // of a row, rows of a warp
        // copied as they are to where they belong, then turned over in place, a thread a row: a row's largest takes no shuffles, which
        // beside the copies' stores are slow (with a row on 16 lanes 11,000 cycles an item, so 7,000)
        const int piece = lane % kLanes;
#pragma unroll 4
        for (int q_row = warp * kAtOnce + lane / kLanes; q_row < tiles * kTileRows; q_row += kSoftmaxWarps * kAtOnce) {
            int head;
            const size_t token = item.span.first + place_of(min(q_row, columns - 1), head);
            const bf16* const from = a.query + token * a.query_stride + (size_t)(item.kv_head * group + head) * HD + piece * 8;
            const uint32_t to = tc::smem_u32(queries) + (q_row / kTileRows) * kTileRows * HD * 2 + tile_offset(q_row % kTileRows, piece);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(q_row < columns ? 16 : 0) : "memory");
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        asm volatile("bar.sync 1, 256;" ::: "memory");
        const int tile = warp >> 2, quarter = warp & 3;
        const int r = tile * kTileRows + quarter * kWarp + lane;
        float up = 0.0f;                                               // of the row's scores
        if (tile < tiles) {
            unsigned char* const row_at = queries + tile * kTileRows * HD * 2;
            int4 raw[kLanes];
            uint32_t most = 0u;
#pragma unroll
            for (int i = 0; i < kLanes; ++i) raw[i] = *reinterpret_cast<const int4*>(row_at + tile_offset(r % kTileRows, i));
#pragma unroll
            for (int i = 0; i < kLanes; ++i) {
                most = __vmaxu2(most, __vmaxu2(__vmaxu2((uint32_t)raw[i].x & 0x7fff7fffu, (uint32_t)raw[i].y & 0x7fff7fffu),
                                               __vmaxu2((uint32_t)raw[i].z & 0x7fff7fffu, (uint32_t)raw[i].w & 0x7fff7fffu)));
            }
            const int shift = query_shift(max(most & 0xffffu, most >> 16));
            const float to_half = power_of_two(shift);
            up = query_back(a.scale * 1.4426950408889634f, shift);
#pragma unroll
            for (int i = 0; i < kLanes; ++i) {
                const uint32_t x[4] = {(uint32_t)raw[i].x, (uint32_t)raw[i].y, (uint32_t)raw[i].z, (uint32_t)raw[i].w};
                uint32_t h[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) h[e] = pack_half2(bf_lo(x[e]) * to_half, bf_hi(x[e]) * to_half);
                *reinterpret_cast<int4*>(row_at + tile_offset(r % kTileRows, i)) = make_int4((int)h[0], (int)h[1], (int)h[2], (int)h[3]);
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&q_ready);
        // ---- softmax: a thread a row
        const bool real = r < columns;
        const int seen = max(seen_by(min(r, columns - 1)) - step0 * kStep, 0);                 // (rows behind the last column: queries of zeros that see what it sees)
        const int unmasked = (int)__reduce_min_sync(0xffffffffu, (unsigned int)seen) / kHalf;      // halves all of which every row of the warp sees
        const uint32_t lanes = tmem + ((uint32_t)(quarter * kWarp) << 16);
        const uint32_t o_at = lanes + kOut + tile * 128;
        const int own = tile < tiles ? halves : 0;
        float top = -INFINITY, total = 0.0f;
        int settled = 0;                                               // halves that every row of the warp sees all of and has a reference for
        auto rescale_output = [&](float keep, int n) {                 // when the products of the halves before are done
            if (!__all_sync(0xffffffffu, guard.wait(&o_ready[tile][(n - 1) & 1], ((n - 1) >> 1) & 1))) return;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
            for (int c = 0; c < HD; c += 16) {
                float o[16];
                uint32_t bits[16];
                tc::tmem_load_row<16>(o_at + c, o);
#pragma unroll
                for (int j = 0; j < 16; ++j) bits[j] = __float_as_uint(o[j] * keep);
                tmem_store_16(o_at + c, bits);
            }
        };
        const bool idle = r - lane >= columns;                         // no row of the warp is real: what stands for its weights is as good as any
        for (int n = 0; idle && n < own; ++n) {
            if (!__all_sync(0xffffffffu, guard.wait(&s_ready[tile][n & 1], (n >> 1) & 1))) break;
            if (lane == 0) tc::mbar_arrive(&p_ready[tile][n & 1]);
        }
        for (int n = idle ? own : 0; n < own; ++n) {
            if (!__all_sync(0xffffffffu, guard.wait(&s_ready[tile][n & 1], (n >> 1) & 1))) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t s_at = lanes + tile * kStep + (n & 1) * kHalf;
            // (read together and ahead: beside the copies' stores and the products' operands a load from shared memory takes 300 cycles)
            float4 page_scales[kHalfPages];
#pragma unroll
            for (int p = 0; p < kHalfPages; ++p) page_scales[p] = scales[(n >> 1) % kScaleRing][(n & 1) * kHalfPages + p];
            uint32_t s[2][32];
            tmem_load_32(s_at, s[0]);
            tmem_load_32(s_at + 32, s[1]);
            tmem_wait_load(s[0]);
            tmem_wait_load(s[1]);
            // No maximum is looked for: a weight is at most its page's sum, which says whether one may have outgrown fp16
            bool written = false;
            if (n < settled) {
                const float reference = top - kKv8Lift;
                uint32_t w[2][16];
                float largest = 0.0f, added = 0.0f;
#pragma unroll
                for (int p = 0; p < kHalfPages; ++p) {
                    const float4 f = page_scales[p];
                    const float slope = f.x * up, shift = f.y - reference;
                    const unsigned long long slope2 = pack2(slope, slope), shift2 = pack2(shift, shift);
                    unsigned long long sums[2];
#pragma unroll
                    for (int j = 0; j < 16; j += 2) {
                        const uint32_t* const at = &s[p >> 1][(p & 1) * 16 + j];
                        float x, y;
                        unpack2(fma2(pack2(__uint_as_float(at[0]), __uint_as_float(at[1])), slope2, shift2), x, y);
                        x = exp2_ftz(x);
                        y = exp2_ftz(y);
                        sums[(j >> 1) & 1] = j < 4 ? pack2(x, y) : add2(sums[(j >> 1) & 1], pack2(x, y));
                        w[p >> 1][(p & 1) * 8 + j / 2] = pack_half2(x, y);
                    }
                    float x, y;
                    unpack2(add2(sums[0], sums[1]), x, y);
                    x += y;
                    largest = fmaxf(largest, x);
                    added = fmaf(x, f.z, added);
                }
                // (nor does this path take value scales below the least)
                static_assert(kHalfPages == 4, "pages of a half");
                if (fminf(fminf(page_scales[0].w, page_scales[1].w), fminf(page_scales[2].w, page_scales[3].w)) != 1.0f) largest = INFINITY;
                if (!__any_sync(0xffffffffu, largest > kMostWeight)) {
                    total += added;
                    tmem_store_16(s_at, w[0]);
                    tmem_store_16(s_at + 16, w[1]);
                    written = true;
                } else {
                    tmem_load_32(s_at, s[0]);
                    tmem_load_32(s_at + 32, s[1]);
                    tmem_wait_load(s[0]);
                    tmem_wait_load(s[1]);
                }
            }
            if (!written) {
                // ---- halves that some row does not see all of, and scores that have outgrown their reference
                const int visible = seen - n * kHalf;                  // of the half's tokens
                float most = -INFINITY;
#pragma unroll
                for (int p = 0; p < kHalfPages; ++p) {
                    float m = -INFINITY;
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        m = fmaxf(m, 16 * p + j >= visible ? -INFINITY : __uint_as_float(s[p >> 1][(p & 1) * 16 + j]));
                    }
                    most = fmaxf(most, m == -INFINITY ? m : fmaf(m, page_scales[p].x * up, page_scales[p].y));
                }
                const float moved = most > top + kKv8Slack ? most : top, keep = moved == top ? 1.0f : exp2_ftz(top - moved);
                top = moved;
                total *= keep;
                if (n > 0 && __any_sync(0xffffffffu, keep != 1.0f)) rescale_output(keep, n);
                settled = __any_sync(0xffffffffu, top == -INFINITY) ? 0 : unmasked;
                // (nothing but -inf so far: weights of zero)
                const float reference = top == -INFINITY ? 0.0f : top - kKv8Lift;
#pragma unroll
                for (int p = 0; p < kHalfPages; ++p) {
                    uint32_t w[8];
                    const float slope = page_scales[p].x * up, shift = page_scales[p].y - reference;
                    float sum = 0.0f;
#pragma unroll
                    for (int j = 0; j < 16; j += 2) {
                        const uint32_t* const at = &s[p >> 1][(p & 1) * 16 + j];
                        const float x = exp2_ftz(16 * p + j >= visible ? -INFINITY : fmaf(__uint_as_float(at[0]), slope, shift));
                        const float y = exp2_ftz(16 * p + j + 1 >= visible ? -INFINITY : fmaf(__uint_as_float(at[1]), slope, shift));
                        sum += x + y;
                        w[j / 2] = pack_half2(x * page_scales[p].w, y * page_scales[p].w);
                    }
                    total = fmaf(sum, page_scales[p].z, total);
                    tmem_store_8(s_at + 8 * p, w);
                }
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&p_ready[tile][n & 1]);
        }
        // (A barrier a half: of the one that is waited for here all completions but the last are known to be past, so that its parity says
        // which.  With one barrier for both halves a late reader would take two completions for none.)
        if (own > 0) guard.wait(&o_ready[tile][(own - 1) & 1], ((own - 1) >> 1) & 1);
        __syncwarp();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const float inverse = parts > 1 ? 1.0f : total == 0.0f ? 0.0f : 1.0f / total;
        float* const part_at = reinterpret_cast<float*>(left + kJointBytes) + (size_t)blockIdx.x * Part<HD>::kFloats;
        int head;
        const size_t token = item.span.first + place_of(min(r, columns - 1), head), at = (size_t)(item.kv_head * group + head) * HD;
        // Rows whose block gave up are left as they were: the mark of a part's, which no row has as its reference, is NaN
        const bool gave_up = __any_sync(0xffffffffu, *abort_flag != 0) || (int)blockIdx.x == lost_block;
        if (parts > 1 && real) *reinterpret_cast<float2*>(part_at + 2 * kTileRows * HD + 2 * r) = make_float2(gave_up ? NAN : top, total);
#pragma unroll 1
        for (int c = 0; c < HD; c += 64) {
            uint32_t o[2][32];
            __syncwarp();                                              // the loads are the whole warp's, what comes before and behind them is not
            if (own > 0) {
                tmem_load_32(o_at + c, o[0]);
                tmem_load_32(o_at + c + 32, o[1]);
                tmem_wait_load(o[0]);
                tmem_wait_load(o[1]);
            }
            if (!real || gave_up) continue;
            // (8 dims)
#pragma unroll
            for (int j = 0; j < 64; j += 8) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = own > 0 ? __uint_as_float(o[j >> 5][(j & 31) + e]) * inverse : 0.0f;
                if (parts > 1) {
                    float4* const to = reinterpret_cast<float4*>(part_at) + (c + j) / 4 * (2 * kTileRows) + r;
                    to[0] = make_float4(v[0], v[1], v[2], v[3]);
                    to[2 * kTileRows] = make_float4(v[4], v[5], v[6], v[7]);
                    continue;
                }
                __nv_bfloat162 x[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
                *reinterpret_cast<int4*>(a.out + token * a.out_stride + at + c + j) = *reinterpret_cast<const int4*>(x);
                if (a.out32 != nullptr) {
                    float* const to = a.out32 + token * a.query_heads * HD + at + c + j;
                    *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
                    *reinterpret_cast<float4*>(to + 4) = make_float4(v[4], v[5], v[6], v[7]);
                }
            }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    }
    __syncwarp();
    __syncthreads();
    if (*abort_flag != 0 || (int)blockIdx.x == lost_block) {
        if (tid == 0) {
            atomicAdd(&g_kv8_prompt_errors, 1u);
            const unsigned long long until = tc::now_ns() + 200000ull;       // products that are still under way
            while (tc::now_ns() < until) __nanosleep(1000);
        }
        __syncthreads();
    }
    if (warp == kProductWarp) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
    }
    pdl_wait();
    pdl_trigger();
}

// An item's parts, one after the other: a CTA 32 of its rows, a warp 8 dims of them at a time.  Rows of which a part is missing are left as they were
template <int HD>
__global__ void __launch_bounds__(256) kv8_join_kernel(const Kv8AttentionArgs a, const int most_parts, const unsigned char* const left) {
    pdl_wait();
    pdl_trigger();
    const int item = (int)blockIdx.x / (2 * kTileRows / kWarp), r = (int)blockIdx.x % (2 * kTileRows / kWarp) * kWarp + (int)threadIdx.x % kWarp;
    const Joint joint = reinterpret_cast<const Joint*>(left)[item];
    if (joint.parts < 2 || r >= joint.columns) return;
    const float* const from = reinterpret_cast<const float*>(left + kJointBytes) + (size_t)item * most_parts * Part<HD>::kFloats;
    const int group = a.query_heads / a.cache.heads, i = (joint.column0 + r) / group;
    const size_t token = joint.first + i, at = (size_t)(joint.kv_head * group + joint.column0 + r - i * group) * HD;
    for (int d = (int)threadIdx.x / kWarp * 8; d < HD; d += 64) {
        Merged v;
        bool missing = false;
#pragma unroll 4
        for (int n = 0; n < joint.parts; ++n) {
            const float* const part = from + n * Part<HD>::kFloats;
            const float4* const o = reinterpret_cast<const float4*>(part) + d / 4 * (2 * kTileRows) + r;
            const float2 stats = *reinterpret_cast<const float2*>(part + 2 * kTileRows * HD + 2 * r);
            missing |= stats.x != stats.x;
            v.add(stats, o[0], o[2 * kTileRows]);
        }
        if (missing) return;
        const float inverse = v.total == 0.0f ? 0.0f : 1.0f / v.total;
        __nv_bfloat162 x[4];
#pragma unroll
        for (int e = 0; e < 8; ++e) v.sum[e] *= inverse;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = __floats2bfloat162_rn(v.sum[2 * e], v.sum[2 * e + 1]);
        *reinterpret_cast<int4*>(a.out + token * a.out_stride + at + d) = *reinterpret_cast<const int4*>(x);
        if (a.out32 != nullptr) {
            float* const to = a.out32 + token * a.query_heads * HD + at + d;
            *reinterpret_cast<float4*>(to) = make_float4(v.sum[0], v.sum[1], v.sum[2], v.sum[3]);
            *reinterpret_cast<float4*>(to + 4) = make_float4(v.sum[4], v.sum[5], v.sum[6], v.sum[7]);
        }
    }
}

// Blocks of 128 columns where 256 would leave SMs idle (one row, 16 query heads on 8, 128 / 256 in us: 1,024 tokens 21 / 27, 2,048 40 / 44, 2,200
// 45 / 46; 3,000, past the rule, 78 / 59), and where those of 256 are so few that each could have several SMs, parts (256 tokens over
// 16,384: 51 us, without 214; over 4,096 32 / 59; over 2,048 31 / 33)
PromptCut prompt_cut(const Kv8AttentionArgs& a) {
    // as many items as any split of the tokens over the rows can make
    const long long columns = (long long)a.tokens * (a.query_heads / a.cache.heads);
    const long long rows = columns / (a.row_columns + 1) < a.rows ? columns / (a.row_columns + 1) : a.rows;
    auto items = [&](int block) {
        return (a.rows == 1 ? (columns + block - 1) / block : columns / block + rows) * a.cache.heads;
    };
    PromptCut cut{2 * kTileRows, 1, items(2 * kTileRows)};
    if (cut.items >= 1 && cut.items <= 148 / 2) {
        const long long parts = 148 / cut.items, most = a.max_sequence / kPartTokens;
        cut.parts = (int)(parts < kMostParts ? parts : kMostParts);
        if (cut.parts > most) cut.parts = (int)most;
    }
    if (cut.parts < 2) {
        cut.parts = 1;
        if ((columns / (2 * kTileRows) + 1) * a.cache.heads <= 148) cut = PromptCut{kTileRows, 1, items(kTileRows)};
    }
    return cut;
}

template <int HD, bool E4M3, bool PARTS>
cudaError_t launch_cut(const Kv8AttentionArgs& a, const PromptCut& cut, unsigned char* left, cudaStream_t stream) {
    static std::atomic<unsigned long long> allowed{0};
    static std::atomic<bool> looked{false};
    if (!looked.load(std::memory_order_acquire)) {
        cudaFuncAttributes built;
        const cudaError_t e = cudaFuncGetAttributes(&built, kv8_prompt_kernel<HD, E4M3, PARTS>);
        if (e != cudaSuccess) return e;
        if (built.numRegs < kLaunchRegisters) return cudaErrorInvalidConfiguration;     // what setmaxnreg hands out has to be there
        looked.store(true, std::memory_order_release);
    }
    const cudaError_t e = kv8_allow_smem(allowed, kv8_prompt_kernel<HD, E4M3, PARTS>, (int)PromptSmem<HD>::kBytes);
    if (e != cudaSuccess) return e;
    const unsigned grid = (unsigned)(cut.items > 0 ? cut.items * cut.parts : 1);
    return launch_pdl(kv8_prompt_kernel<HD, E4M3, PARTS>, dim3(grid), dim3(kPromptThreads), PromptSmem<HD>::kBytes, stream, a, cut.block_columns, cut.parts, left,
                      g_lost_block.load(std::memory_order_relaxed));
}

template <int HD, bool E4M3>
cudaError_t launch_prompts(const Kv8AttentionArgs& a, cudaStream_t stream) {
    const PromptCut cut = prompt_cut(a);
    if (cut.items > 0x7fffffffll) return cudaErrorInvalidValue;
    unsigned char* const left = static_cast<unsigned char*>(a.scratch) + a.scratch_taken;
    if (cut.parts < 2) return launch_cut<HD, E4M3, false>(a, cut, left, stream);
    const cudaError_t e = launch_cut<HD, E4M3, true>(a, cut, left, stream);
    return e != cudaSuccess ? e : launch_pdl(kv8_join_kernel<HD>, dim3((unsigned)cut.items * (2 * kTileRows / kWarp)), dim3(256), 0, stream, a, cut.parts, left);
}

}  // namespace

size_t kv8_prompt_scratch_bytes(int max_sequence, int head_dim) {
    return max_sequence < 2 * kPartTokens ? 0 : kJointBytes + 148 * (head_dim == 128 ? Part<128>::kFloats : Part<64>::kFloats) * sizeof(float);
}

cudaError_t launch_kv8_prompts(const Kv8AttentionArgs& a, int head_dim, bool e4m3, cudaStream_t stream) {
    if (head_dim == 128) return e4m3 ? launch_prompts<128, true>(a, stream) : launch_prompts<128, false>(a, stream);
    return e4m3 ? launch_prompts<64, true>(a, stream) : launch_prompts<64, false>(a, stream);
}

void lose_kv8_block(int block) { g_lost_block.store(block, std::memory_order_relaxed); }

unsigned int kv8_prompt_error_count() {
    unsigned int v = 0;
    return cudaMemcpyFromSymbol(&v, g_kv8_prompt_errors, sizeof(v)) == cudaSuccess ? v : ~0u;
}
unsigned int kv8_prompt_range_error_count() {
    unsigned int v = 0;
    return cudaMemcpyFromSymbol(&v, g_kv8_prompt_range_errors, sizeof(v)) == cudaSuccess ? v : ~0u;
}
unsigned int kv8_prompt_page_error_count() {
    unsigned int v = 0;
    return cudaMemcpyFromSymbol(&v, g_kv8_prompt_page_errors, sizeof(v)) == cudaSuccess ? v : ~0u;
}

}  // namespace q3t
