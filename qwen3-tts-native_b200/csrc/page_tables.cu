// Block tables, positions and slot maps of a batch, built on the GPU from the requests' lengths (q3t_launch_page_tables).
//
// Row r of length n and change c needs ceil((n + c) / 16) - ceil(n / 16) pages when it grows and gives that many back when it
// shrinks.  All pages given back go onto the stack first, then rows that grow take theirs from its top, both in the order of
// the rows, so three prefix sums say everything: the k-th page taken is the entry at (available - 1 - k), which lies in
// the old stack or, above its top, in the table of a row that gives back, found by a search in its prefix sum.  No page is moved
// through memory to be taken in the same launch, and nothing is serial in the rows.
//
// What bounds it: latency (lengths, sums, table entries: three loads one behind the other) and, with long prompts, the 12 bytes
// a new token that are written.  Every CTA repeats the sums, which are cheap beside a second launch; a barrier over the
// cluster separates the last read of lengths and free_count from the first write of what may be the same memory.

#include "kv8.cuh"
#include "q3t_kernels.cuh"

#include <climits>

namespace q3t {
namespace {

constexpr int kTableThreads = 1024;
constexpr int kTableWarps = kTableThreads / kWarp;
constexpr int kTableCluster = 8;               // CTAs for more tokens than one writes at once
constexpr int kRowsPerThread = Q3T_MAX_TABLE_ROWS / kTableThreads;
constexpr int kTokensPerThread = 4;            // consecutive, of mostly one row and one page

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

// exclusive prefix sums over the threads of the block; `total` gets the sums over all of them
template <class T, int N>
__device__ __forceinline__ void block_scan(T (&v)[N], T (&total)[N], T* warp_sums) {
    const int lane = threadIdx.x % kWarp, warp = threadIdx.x / kWarp;
    T mine[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        mine[i] = v[i];
#pragma unroll
        for (int o = 1; o < kWarp; o <<= 1) {
            const T other = __shfl_up_sync(0xffffffffu, v[i], o);
            if (lane >= o) v[i] += other;
        }
        if (lane == kWarp - 1) warp_sums[i * kTableWarps + warp] = v[i];
        v[i] -= mine[i];
    }
    __syncthreads();
    if (warp < N) {
        const T own = warp_sums[warp * kTableWarps + lane];
        T sum = own;
#pragma unroll
        for (int o = 1; o < kWarp; o <<= 1) {
            const T other = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += other;
        }
        warp_sums[warp * kTableWarps + lane] = sum - own;
        if (lane == kWarp - 1) warp_sums[N * kTableWarps + warp] = sum;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] += warp_sums[i * kTableWarps + warp];
        total[i] = warp_sums[N * kTableWarps + i];
    }
    __syncthreads();
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

__global__ void __launch_bounds__(kTableThreads) page_tables_kernel(const TableArgs a) {
    extern __shared__ int smem[];
    int* const token_start = smem;                     // [rows] of the tokens that are served
    int* const need_start = token_start + a.rows;      // [rows] of the pages taken, clamped
    int* const given_start = need_start + a.rows;      // [rows] of the pages given back, clamped
    int* const aside = given_start + a.rows;           // [rows] growing: its length; shrinking: the pages it keeps
    __shared__ long long warp_sums[3 * kTableWarps + 3];
    static_assert(kPageTokens == 16, "pages_of");

    unsigned int rank, ctas;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
    const int tid = threadIdx.x;
    pdl_wait();
    pdl_trigger();

    // ---- the sums
    const int per = (a.rows + kTableThreads - 1) / kTableThreads;      // at most kRowsPerThread
    const int first = tid * per;
    int length[kRowsPerThread], change[kRowsPerThread];
    long long sums[3] = {0, 0, 0};                     // tokens asked for, pages asked for, pages given back
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) {
        const int row = first + i;
        const bool mine = i < per && row < a.rows;
        length[i] = mine ? a.lengths[row] : 0;
        change[i] = mine ? a.changes[row] : 0;
    }
    const int free = min(max(*a.free_count, 0), a.pages);
    const long long room = (long long)a.stride * kPageTokens;
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) {
        const long long want = (long long)length[i] + change[i];
        if (length[i] < 0 || length[i] > room || want < 0 || want > room) {
            length[i] = INT_MIN;                       // refused
            continue;
        }
        const int pages = pages_of((int)want) - pages_of(length[i]);
        if (change[i] > 0) {
            sums[0] += change[i];
            sums[1] += pages;
        } else {
            sums[2] -= pages;
        }
    }
    long long total[3];
    block_scan(sums, total, warp_sums);
    // ids beyond what the stack has room for are dropped
    const int available = (int)min((long long)free + total[2], (long long)a.pages);
    int served[2] = {0, 0};                            // tokens, pages
    int state[kRowsPerThread];
    {
        long long asked = sums[0], need = sums[1];
#pragma unroll
        for (int i = 0; i < kRowsPerThread; ++i) {
            state[i] = Q3T_TABLE_OK;
            if (length[i] == INT_MIN) state[i] = Q3T_TABLE_LENGTH;
            else if (change[i] > 0) {
                const int pages = pages_of(length[i] + change[i]) - pages_of(length[i]);
                asked += change[i];
                need += pages;
                if (asked > a.capacity) state[i] = Q3T_TABLE_NO_TOKENS;
                else if (pages > 0 && need > available) state[i] = Q3T_TABLE_NO_PAGES;
                else {
                    served[0] += change[i];
                    served[1] += pages;
                }
            }
        }
    }
    int all[2];
    block_scan(served, all, reinterpret_cast<int*>(warp_sums));
    {
        int tokens = served[0];
        long long need = sums[1], given = sums[2];
#pragma unroll
        for (int i = 0; i < kRowsPerThread; ++i) {
            const int row = first + i;
            if (i >= per || row >= a.rows) break;
            token_start[row] = tokens;
            need_start[row] = (int)min(need, (long long)INT_MAX);
            given_start[row] = (int)min(given, (long long)INT_MAX);
            aside[row] = length[i];
            if (length[i] == INT_MIN) continue;
            const int before = pages_of(length[i]), after = pages_of(length[i] + change[i]);
            if (change[i] > 0) {
                need += after - before;
                if (state[i] == Q3T_TABLE_OK) tokens += change[i];
            } else {
                given += before - after;
                aside[row] = after;
            }
        }
    }
    // from here on lengths and free_count may be written
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    __syncthreads();
    const int tokens = all[0], taken = all[1];
    if (rank == 0) {
#pragma unroll
        for (int i = 0; i < kRowsPerThread; ++i) {
            const int row = first + i;
            if (i >= per || row >= a.rows) break;
            a.status[row] = state[i];
            a.starts[row] = token_start[row];
            if (state[i] == Q3T_TABLE_OK) a.new_lengths[row] = length[i] + change[i];
            else if (a.new_lengths != a.lengths) a.new_lengths[row] = a.lengths[row];
        }
        if (tid == 0) {
            a.starts[a.rows] = tokens;
            *a.new_free_count = available - taken;
        }
    }

    // the id at a place of the stack once everything is given back
    auto id_at = [&](int place) {
        if (place < free) return a.stack[place];
        const int given = place - free, row = row_of(given_start, a.rows, given);
        return a.table[(size_t)row * a.stride + aside[row] + given - given_start[row]];
    };
    const int threads = (int)ctas * kTableThreads, thread = (int)rank * kTableThreads + tid;
    // ---- pages given back that stay on the stack, pages taken
    for (int place = free + thread; place < available - taken; place += threads) a.stack[place] = id_at(place);
    for (int k = thread; k < taken; k += threads) {
        const int row = row_of(need_start, a.rows, k);
        a.table[(size_t)row * a.stride + pages_of(aside[row]) + k - need_start[row]] = id_at(available - 1 - k);
    }
    // ---- tokens
    if (a.positions == nullptr && a.slots == nullptr) return;
    for (long long t0 = (long long)thread * kTokensPerThread; t0 < tokens; t0 += (long long)threads * kTokensPerThread) {
        int row = row_of(token_start, a.rows, (int)t0), page = -1, id = 0;
#pragma unroll
        for (int i = 0; i < kTokensPerThread; ++i) {
            const int t = (int)t0 + i;
            if (t >= tokens) break;
            while (row + 1 < a.rows && token_start[row + 1] <= t) {
                ++row;
                page = -1;
            }
            const int position = aside[row] + t - token_start[row];
            if (a.positions != nullptr) a.positions[t] = position;
            if (a.slots == nullptr) continue;
            if (position / kPageTokens != page) {
                page = position / kPageTokens;
                const int fresh = page - pages_of(aside[row]);
                id = fresh < 0 ? a.table[(size_t)row * a.stride + page] : id_at(available - 1 - (need_start[row] + fresh));
            }
            a.slots[t] = (long long)id * kPageTokens + position % kPageTokens;
        }
    }
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
    const size_t smem = (size_t)d->rows * 4 * sizeof(int);
    static std::atomic<unsigned long long> allowed{0};
    if (const cudaError_t e = kv8_allow_smem(allowed, page_tables_kernel, Q3T_MAX_TABLE_ROWS * 4 * (int)sizeof(int))) return e;
    TableArgs a;
    a.lengths = d->lengths; a.changes = d->changes; a.new_lengths = d->new_lengths; a.table = d->page_table;
    a.stack = d->free_pages; a.free_count = d->free_count; a.new_free_count = d->new_free_count; a.status = d->status;
    a.starts = d->token_starts; a.positions = d->positions; a.slots = reinterpret_cast<long long*>(d->slots);
    a.rows = d->rows; a.stride = d->page_table_stride; a.pages = d->pages; a.capacity = d->token_capacity;
    cudaLaunchConfig_t cfg = {};
    const unsigned ctas = d->token_capacity > kTableThreads * kTokensPerThread ? kTableCluster : 1;
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kTableThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return static_cast<int32_t>(cudaLaunchKernelEx(&cfg, page_tables_kernel, a));
}
