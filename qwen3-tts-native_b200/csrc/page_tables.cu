// Block tables, positions and slot maps of a batch, built on the GPU from the requests' lengths (q3t_launch_page_tables).
//
// Row r of length n and change c needs ceil((n + c) / 16) - ceil(n / 16) pages when it grows and gives that many back when it
// shrinks.  All pages given back go onto the stack first, then rows that grow take theirs from its top, both in the order of
// the rows, so three prefix sums say everything: the k-th page taken is the entry at (available - 1 - k), which lies in
// the old stack or, above its top, in the table of a row that gives back, found by a search in its prefix sum.  No page is moved
// through memory to be taken in the same launch, and nothing is serial in the rows.
//
// What bounds it: latency (lengths, sums, table entries: three loads one behind the other) and, with long prompts, the 12 bytes
// a new token that are written.  A step of a token a row is one CTA's.  Others are filled in by a CTA for each 32 rows or 2,048 tokens, each of
// which repeats the sums, and a second launch writes lengths, states and the free count, which may lie over what the first one
// reads (where they do not, its first CTA could write them: not done); it has its sums by the time the first is done.  One CTA / two
// launches, in us: a token a row 3.2 / 3.8 (64 rows), 4.3 / 4.7 (512), 6.3 / 5.5
// (1,000); every eighth row with a prompt of up to 8 tokens and every sixteenth giving all pages back 7.0 / 6.5 (64), 13.2 / 8.7 (1,000); prompts of
// up to 1,500 for 113,000 tokens 69.6 / 8.7 (1.4 MB written, 0.3 us of memory).

#include "kv8.cuh"
#include "q3t_kernels.cuh"

#include <climits>

namespace q3t {
namespace {

constexpr int kMostThreads = 1024;
constexpr int kFillThreads = 512;              // of the CTAs that only fill in
constexpr int kChunk = 128;                    // tokens, or pages given back, that a warp takes at a time
constexpr int kFew = 8;                        // tokens of a row that a thread fills in
constexpr int kOneCtaRows = 512;
constexpr int kCtaTokens = kFillThreads / kWarp * kChunk, kCtaRows = 32;      // of a CTA that fills in
constexpr int kFill = 1, kSettle = 2;          // what a launch writes: tables, stack and tokens; lengths, states, starts and the free count

struct TableArgs {
    const int* lengths;
    const int* changes;
    int* new_lengths;
    int* table;
    int* stack;
    const int* free_count;
    int* new_free_count;
    int* status;
    int* starts;
    int* positions;
    long long* slots;
    int rows, stride, pages, capacity;
};

// sums that stop at 2^32 - 1, which is more than any of them is compared with
__device__ __forceinline__ unsigned int add_up(unsigned int a, unsigned int b) {
    const unsigned int sum = a + b;
    return sum < a ? ~0u : sum;
}

// prefix sums over the threads of the block, ahead of each and of all
template <int N>
__device__ __forceinline__ void block_scan(unsigned int (&v)[N], unsigned int (&total)[N], unsigned int (*warp_sums)[kWarp]) {
    const int lane = threadIdx.x % kWarp, warp = threadIdx.x / kWarp, warps = (int)blockDim.x / kWarp;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        unsigned int sum = v[i];
#pragma unroll
        for (int o = 1; o < kWarp; o <<= 1) {
            const unsigned int other = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum = add_up(sum, other);
        }
        if (lane == kWarp - 1) warp_sums[i][warp] = sum;
        const unsigned int ahead = __shfl_up_sync(0xffffffffu, sum, 1);
        v[i] = lane > 0 ? ahead : 0u;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        // every warp adds up the warps' sums for itself
        unsigned int sum = lane < warps ? warp_sums[i][lane] : 0u;
#pragma unroll
        for (int o = 1; o < kWarp; o <<= 1) {
            const unsigned int other = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum = add_up(sum, other);
        }
        total[i] = __shfl_sync(0xffffffffu, sum, kWarp - 1);
        const unsigned int ahead = __shfl_sync(0xffffffffu, sum, max(warp - 1, 0));
        v[i] = add_up(v[i], warp > 0 ? ahead : 0u);
    }
}

// the last row whose prefix sum is at most `value`
__device__ __forceinline__ int row_of(const int* starts, int rows, int value) {
    int low = 0, high = rows - 1;
    while (low < high) {
        const int middle = (low + high + 1) >> 1;
        if (starts[middle] <= value) low = middle;
        else high = middle - 1;
    }
    return low;
}

__device__ __forceinline__ int pages_of(int tokens) { return (tokens >> 4) + ((tokens & 15) != 0 ? 1 : 0); }

// a row's length and change, and what they come to
struct RowChange {
    int length, change, before, after;         // pages
    bool legal;
    __device__ __forceinline__ RowChange(const TableArgs& a, int length_now, int change_now) : length(length_now), change(change_now) {
        const long long room = (long long)a.stride * kPageTokens, want = (long long)length + change;
        legal = length >= 0 && length <= room && want >= 0 && want <= room;
        before = legal ? pages_of(length) : 0;
        after = legal ? pages_of((int)want) : 0;
    }
    __device__ __forceinline__ bool grows() const { return legal && change > 0; }
    __device__ __forceinline__ unsigned int asked() const { return grows() ? (unsigned int)change : 0u; }
    __device__ __forceinline__ unsigned int need() const { return grows() ? (unsigned int)(after - before) : 0u; }
    // of a row that is served: its tokens unless they are few, or the pages that it gives back
    __device__ __forceinline__ unsigned int chunks() const {
        return change > 0 ? (change <= kFew ? 0u : (asked() + kChunk - 1) / kChunk) : (given() + kChunk - 1) / kChunk;
    }
    __device__ __forceinline__ unsigned int given() const { return legal && change < 0 ? (unsigned int)(before - after) : 0u; }
};

template <int WRITES>
__global__ void __launch_bounds__(WRITES == kFill ? kFillThreads : kMostThreads) page_tables_kernel(const TableArgs a) {
    extern __shared__ int smem[];
    int* const token_start = smem;                     // [rows] of the tokens that are served
    int* const need_start = token_start + a.rows;      // [rows] of the pages taken
    int* const given_start = need_start + a.rows;      // [rows] of the pages given back
    int* const aside = given_start + a.rows;           // [rows] growing: its length; shrinking: the pages it keeps
    int* const chunk_start = aside + a.rows;           // [rows] of what warps do
    int* const lengths = token_start;                  // until a row's sums take their place
    int* const changes = need_start;
    __shared__ unsigned int warp_sums[2][3][kWarp];    // (of two scans: one barrier fewer)
    static_assert(kPageTokens == 16, "pages_of");
    const int tid = threadIdx.x, lane = tid % kWarp, threads_here = (int)blockDim.x;
    if (WRITES != kSettle) {                           // (the launch ahead of that one is the filling one's, which has waited)
        pdl_wait();
        pdl_trigger();
    }

    // ---- the sums
    for (int row = tid; row < a.rows; row += threads_here) {
        lengths[row] = a.lengths[row];
        changes[row] = a.changes[row];
    }
    const int free = min(max(*a.free_count, 0), a.pages);
    __syncthreads();
    const int per = (a.rows + threads_here - 1) / threads_here, first = min(tid * per, a.rows), last = min(first + per, a.rows);
    unsigned int sums[3] = {0u, 0u, 0u}, all[3];       // tokens asked for, pages asked for, pages given back
    for (int row = first; row < last; ++row) {
        const RowChange c(a, lengths[row], changes[row]);
        sums[0] = add_up(sums[0], c.asked());
        sums[1] = add_up(sums[1], c.need());
        sums[2] = add_up(sums[2], c.given());
    }
    block_scan(sums, all, warp_sums[0]);
    // ids beyond what the stack has room for are dropped
    const int available = (int)min((unsigned long long)free + all[2], (unsigned long long)a.pages);
    unsigned int served[3] = {0u, 0u, 0u}, made[3];    // tokens, pages, chunks
    auto state_of = [&](const RowChange& c, unsigned int asked, unsigned int need) {       // the sums with this row's own
        return !c.legal ? Q3T_TABLE_LENGTH : c.change <= 0 ? Q3T_TABLE_OK : asked > (unsigned int)a.capacity ? Q3T_TABLE_NO_TOKENS
               : c.need() > 0u && need > (unsigned int)available ? Q3T_TABLE_NO_PAGES : Q3T_TABLE_OK;
    };
    unsigned int asked = sums[0], need = sums[1], given = sums[2];
    for (int row = first; row < last; ++row) {
        const RowChange c(a, lengths[row], changes[row]);
        asked = add_up(asked, c.asked());
        need = add_up(need, c.need());
        if (state_of(c, asked, need) == Q3T_TABLE_OK) {
            served[0] += c.asked();
            served[1] += c.need();
            served[2] += c.chunks();
        }
    }
    block_scan(served, made, warp_sums[1]);
    const int tokens = (int)made[0], taken = (int)made[1], chunks = (int)made[2];
    asked = sums[0];
    need = sums[1];
    for (int row = first; row < last; ++row) {
        const RowChange c(a, lengths[row], changes[row]);
        token_start[row] = (int)served[0];
        need_start[row] = (int)min(need, (unsigned int)INT_MAX);
        given_start[row] = (int)min(given, (unsigned int)INT_MAX);
        aside[row] = c.change > 0 ? c.length : c.after;
        chunk_start[row] = (int)served[2];
        asked = add_up(asked, c.asked());
        need = add_up(need, c.need());
        given = add_up(given, c.given());
        const int state = state_of(c, asked, need);
        if (state == Q3T_TABLE_OK) {
            served[0] += c.asked();
            served[2] += c.chunks();
        }
        if (WRITES == kSettle) pdl_wait();             // the filling launch reads lengths and free_count
        if (WRITES & kSettle) {
            a.status[row] = state;
            a.starts[row] = token_start[row];
            a.new_lengths[row] = state == Q3T_TABLE_OK ? c.length + c.change : c.length;
        }
    }
    __syncthreads();
    if (WRITES == kSettle) {
        pdl_wait();
        pdl_trigger();
    }
    if ((WRITES & kSettle) && tid == 0) {
        a.starts[a.rows] = tokens;
        *a.new_free_count = available - taken;
    }
    if (WRITES == kSettle) return;

    // the id at a place of the stack once everything is given back
    auto id_at = [&](int place) {
        if (place < free) return a.stack[place];
        const int n = place - free, row = row_of(given_start, a.rows, n);
        return a.table[(size_t)row * a.stride + aside[row] + n - given_start[row]];
    };
    auto id_of = [&](int row, int page) {
        const int fresh = page - pages_of(aside[row]);
        return fresh < 0 ? a.table[(size_t)row * a.stride + page] : id_at(available - 1 - (need_start[row] + fresh));
    };
    auto write = [&](int t, int position, int id) {
        if (a.positions != nullptr) a.positions[t] = position;
        if (a.slots != nullptr) a.slots[t] = (long long)id * kPageTokens + position % kPageTokens;
    };
    const int threads = (int)gridDim.x * threads_here, thread = (int)blockIdx.x * threads_here + tid;
    // ---- rows of few tokens, a thread each
    for (int row = thread; row < a.rows; row += threads) {
        const int t0 = token_start[row], count = (row + 1 < a.rows ? token_start[row + 1] : tokens) - t0;
        if (count < 1 || count > kFew) continue;
        const int from = aside[row];
        for (int n = 0; n < count;) {
            const int page = (from + n) / kPageTokens, id = id_of(row, page);
            if ((from + n) % kPageTokens == 0) a.table[(size_t)row * a.stride + page] = id;
            for (; n < count && (from + n) / kPageTokens == page; ++n) write(t0 + n, from + n, id);
        }
    }
    // ---- the others, a warp a chunk
    for (int chunk = thread / kWarp; chunk < chunks; chunk += threads / kWarp) {
        const int row = row_of(chunk_start, a.rows, chunk), skip = (chunk - chunk_start[row]) * kChunk;
        const int t0 = token_start[row], count = (row + 1 < a.rows ? token_start[row + 1] : tokens) - t0;
        if (count > 0) {
            // tokens: an id a lane; the page's first token writes it into the table where it is new
            const int from = aside[row] + skip, here = min(kChunk, count - skip), page0 = from / kPageTokens;
            int id = 0;
            if (lane <= (from + here - 1) / kPageTokens - page0) {
                id = id_of(row, page0 + lane);
                if ((page0 + lane) * kPageTokens >= from) a.table[(size_t)row * a.stride + page0 + lane] = id;
            }
#pragma unroll
            for (int i = 0; i < kChunk / kWarp; ++i) {
                const int n = i * kWarp + lane;
                const int own = __shfl_sync(0xffffffffu, id, min((from + n) / kPageTokens - page0, kWarp - 1));
                if (n < here) write(t0 + skip + n, from + n, own);
            }
        } else {
            // pages given back: those that stay on the stack
            const int given_here = (row + 1 < a.rows ? given_start[row + 1] : (int)min(all[2], (unsigned int)INT_MAX)) - given_start[row];
            for (int n = skip + lane; n < min(skip + kChunk, given_here); n += kWarp) {
                const long long place = (long long)free + given_start[row] + n;
                if (place < available - taken) a.stack[place] = a.table[(size_t)row * a.stride + aside[row] + n];
            }
        }
    }
}

template <int WRITES>
cudaError_t launch_tables(const TableArgs& a, int ctas, int threads, cudaStream_t stream) {
    const int smem = a.rows * 5 * (int)sizeof(int);
    static std::atomic<unsigned long long> allowed{0};
    const cudaError_t e = kv8_allow_smem(allowed, page_tables_kernel<WRITES>, Q3T_MAX_TABLE_ROWS * 5 * (int)sizeof(int));
    return e != cudaSuccess ? e : launch_pdl(page_tables_kernel<WRITES>, dim3((unsigned)ctas), dim3((unsigned)threads), (size_t)smem, stream, a);
}

}  // namespace
}  // namespace q3t

extern "C" int32_t q3t_launch_page_tables(const Q3tPageTablesDesc* d, void* stream) {
    using namespace q3t;
    if (d == nullptr || d->struct_size != sizeof(Q3tPageTablesDesc) || d->rows < 1 || d->rows > Q3T_MAX_TABLE_ROWS
        || d->lengths == nullptr || d->changes == nullptr || d->new_lengths == nullptr || d->page_table == nullptr
        || d->free_pages == nullptr || d->free_count == nullptr || d->new_free_count == nullptr || d->status == nullptr
        || d->token_starts == nullptr || d->page_table_stride < 1 || d->page_table_stride > INT_MAX / kPageTokens
        || d->pages < 1 || d->token_capacity < 0 || d->reserved != 0) {
        return cudaErrorInvalidValue;
    }
    TableArgs a;
    a.lengths = d->lengths; a.changes = d->changes; a.new_lengths = d->new_lengths; a.table = d->page_table;
    a.stack = d->free_pages; a.free_count = d->free_count; a.new_free_count = d->new_free_count; a.status = d->status;
    a.starts = d->token_starts; a.positions = d->positions; a.slots = reinterpret_cast<long long*>(d->slots);
    a.rows = d->rows; a.stride = d->page_table_stride; a.pages = d->pages; a.capacity = d->token_capacity;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int rows_up = (d->rows + kWarp - 1) / kWarp * kWarp;
    if (d->token_capacity <= d->rows && d->rows <= kOneCtaRows) return static_cast<int32_t>(launch_tables<kFill | kSettle>(a, 1, rows_up, s));
    const int for_tokens = d->token_capacity / kCtaTokens + 1, for_rows = (d->rows + kCtaRows - 1) / kCtaRows;
    const int ctas = for_tokens > for_rows ? for_tokens : for_rows;
    const cudaError_t e = launch_tables<kFill>(a, ctas < 148 ? ctas : 148, kFillThreads, s);
    return static_cast<int32_t>(e != cudaSuccess ? e : launch_tables<kSettle>(a, 1, rows_up < kMostThreads ? rows_up : kMostThreads, s));
}
