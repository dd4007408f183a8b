// Block tables, row maps and slot maps of one step of continuous batching, from
// request lengths, in one launch without a copy to the host.
//
// Sequence i holds ctx[i] tokens in the paged cache and brings add[i] more.
//   starts = exclusive prefix sum of add           first packed row of each sequence
//   have_i = ceil(ctx_i / 64), need_i = ceil((ctx_i + add_i) / 64)
//   base   = exclusive prefix sum of need - have   its place in the free list
//   table[i][have_i + j] = free[base_i + j]        for the need_i - have_i new pages
//   row r of sequence i: pos = ctx_i + r - starts_i, slot = 64 table[i][pos / 64] + pos % 64
//
// A step writes 16 bytes for each row of rows_cap, the -1 behind the last row
// included (117 KB for 7.3 k rows), so latency bounds it unless rows_cap is far
// beyond the step: one launch, and every CTA computes the prefix sums of all sequences
// itself (8 bytes each, from L2) instead of waiting for another CTA.  A row
// reads table entries below have_i only, and the launch writes entries from
// have_i on only, so the CTAs need no order among themselves.  A step of 64
// sequences, or 512 of 16 to 600 tokens, takes 5.9 us by itself and 3.1 us in a
// captured graph, of which the empty launch is most.
#include "common.cuh"
#include "wukong_ext.h"
#include "wukong_internal.cuh"

namespace wk {

namespace {

constexpr int kPlanPage = 64;
constexpr int kPlanThreads = 256;
constexpr int kPlanMaxSeqs = 8192;  // prefix sums of all sequences in shared memory (16 bytes each)

struct PlanArgs {
    int *starts, *lens, *row_seq, *row_pos;
    long long *row_slot;
    int rows_cap;
    int *table;
    int max_pages;
    int *status;
    const int *ctx, *add;
    int n;
    const int *free_pages, *n_free;
    int free_cap;
};

// The last index i in [0, n) with a[i] <= v (a ascending, a[0] <= v).
__device__ __forceinline__ int last_le(const int *a, int n, int v) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= v)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(kPlanThreads) batch_plan_kernel(PlanArgs a) {
    extern __shared__ int plan_sm[];
    int *s_start = plan_sm;             // [n + 1] first row of each sequence
    int *s_base = s_start + a.n + 1;    // [n + 1] its place in the free list
    int *s_ctx = s_base + a.n + 1;      // [n]
    int *s_add = s_ctx + a.n;           // [n]
    __shared__ long long s_rows[kPlanThreads / 32];
    __shared__ int s_new[kPlanThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    pdl_wait();
    pdl_trigger();
    for (int i = tid; i < a.n; i += kPlanThreads) {
        s_ctx[i] = max(a.ctx[i], 0);
        s_add[i] = max(a.add[i], 0);
    }
    const int n_free = min(max(*a.n_free, 0), a.free_cap);
    __syncthreads();
    // thread t sums sequences [t per, t per + per); scan over the threads
    const int per = (a.n + kPlanThreads - 1) / kPlanThreads;
    const int i0 = min(a.n, tid * per), i1 = min(a.n, i0 + per);
    auto pages = [&](long long tokens) -> int {
        const long long p = (tokens + kPlanPage - 1) / kPlanPage;
        return (int)(p < a.max_pages ? p : a.max_pages);
    };
    long long rows = 0;  // 64 bits: the sum of any lengths
    int fresh = 0;
    for (int i = i0; i < i1; ++i) {
        rows += s_add[i];
        fresh += pages((long long)s_ctx[i] + s_add[i]) - pages(s_ctx[i]);
    }
    long long rows_in = rows;
    int fresh_in = fresh;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long r = __shfl_up_sync(0xffffffffu, rows_in, o);
        const int f = __shfl_up_sync(0xffffffffu, fresh_in, o);
        if (lane >= o) {
            rows_in += r;
            fresh_in += f;
        }
    }
    if (lane == 31) {
        s_rows[wid] = rows_in;
        s_new[wid] = fresh_in;
    }
    __syncthreads();
    long long row0 = rows_in - rows;
    int new0 = fresh_in - fresh;
    for (int w = 0; w < wid; ++w) {
        row0 += s_rows[w];
        new0 += s_new[w];
    }
    auto sat = [](long long v) -> int { return (int)(v < 0x7fffffffll ? v : 0x7fffffffll); };
    for (int i = i0; i < i1; ++i) {
        s_start[i] = sat(row0);
        s_base[i] = new0;
        row0 += s_add[i];
        new0 += pages((long long)s_ctx[i] + s_add[i]) - pages(s_ctx[i]);
    }
    if (tid == kPlanThreads - 1) {  // the last thread's running sums are the totals
        s_start[a.n] = sat(row0);
        s_base[a.n] = new0;
    }
    __syncthreads();
    const int total = s_start[a.n], taken = s_base[a.n];
    // (unsigned: rows_cap and the new pages reach 2^31 - 1, and a step beyond them must not come out negative)
    const unsigned g0 = blockIdx.x * kPlanThreads + tid, gn = gridDim.x * kPlanThreads;
    // rows
    for (unsigned x = g0; x < (unsigned)a.rows_cap; x += gn) {
        const int r = (int)x;
        int seq = -1, pos = -1;
        long long slot = -1;
        if (r < total) {
            seq = last_le(s_start, a.n, r);
            const long long p = (long long)s_ctx[seq] + (r - s_start[seq]);
            pos = sat(p);
            const long long pi = p / kPlanPage;
            if (pi < a.max_pages) {
                const int have = pages(s_ctx[seq]);
                int page;
                if (pi < have) {
                    page = a.table[(long)seq * a.max_pages + pi];
                } else {
                    const int j = s_base[seq] + (int)(pi - have);
                    page = j < n_free ? a.free_pages[j] : -1;
                }
                if (page >= 0) slot = (long long)page * kPlanPage + p % kPlanPage;
            }
        }
        a.row_seq[r] = seq;
        a.row_pos[r] = pos;
        if (a.row_slot) a.row_slot[r] = slot;
    }
    // new table entries
    for (unsigned x = g0; x < (unsigned)taken; x += gn) {
        const int j = (int)x;
        const int seq = last_le(s_base, a.n, j);
        a.table[(long)seq * a.max_pages + pages(s_ctx[seq]) + (j - s_base[seq])] = j < n_free ? a.free_pages[j] : -1;
    }
    // per sequence
    for (unsigned i = g0; i < (unsigned)a.n; i += gn) {
        a.starts[i] = s_start[i];
        a.lens[i] = sat((long long)s_ctx[i] + s_add[i]);
    }
    if (g0 == 0) {
        a.starts[a.n] = total;
        a.status[0] = total;
        a.status[1] = min(taken, n_free);
        a.status[2] = taken - min(taken, n_free);
    }
}

}  // namespace

}  // namespace wk

using namespace wk;

extern "C" {

int wk_batch_plan(int *starts, int *lens, int *row_seq, int *row_pos, long long *row_slot, int rows_cap,
                  int *block_table, int max_pages, int *status, const int *ctx, const int *add, int n,
                  const int *free_pages, const int *n_free, int free_cap) {
    if (n < 1 || n > kPlanMaxSeqs) return fail("wk_batch_plan: n %d (1..%d)", n, kPlanMaxSeqs);
    if (rows_cap < 0 || max_pages < 1 || free_cap < 0) return fail("wk_batch_plan: bad sizes");
    if ((long long)n * max_pages > 0x7fffffffll) return fail("wk_batch_plan: n * max_pages above 2^31 - 1");
    if (!starts || !lens || !block_table || !status || !ctx || !add || !n_free || (rows_cap && (!row_seq || !row_pos)) ||
        (free_cap && !free_pages))
        return fail("wk_batch_plan: null argument");
    const uintptr_t low = (uintptr_t)starts | (uintptr_t)lens | (uintptr_t)row_seq | (uintptr_t)row_pos |
                          (uintptr_t)block_table | (uintptr_t)status | (uintptr_t)ctx | (uintptr_t)add |
                          (uintptr_t)free_pages | (uintptr_t)n_free;
    if (low % 4 || (uintptr_t)row_slot % 8) return fail("wk_batch_plan: misaligned argument");
    if (lens == ctx || lens == add || starts == ctx || starts == add)
        return fail("wk_batch_plan: starts and lens must not be the arrays of the lengths");
    if (g_rt.device < 0) return fail("wk_batch_plan: cuda_init() has not been called");
    DeviceGuard guard;
    PlanArgs a{starts, lens, row_seq, row_pos, row_slot, rows_cap, block_table, max_pages,
               status, ctx,  add,     n,       free_pages, n_free, free_cap};
    const size_t smem = sizeof(int) * (4 * (size_t)n + 2);
    static int configured = -1;  // the device that the kernel is set up for
    if (smem > 48 * 1024 && configured != g_rt.device) {
        cudaError_t e = cudaFuncSetAttribute(batch_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)(sizeof(int) * (4 * (size_t)kPlanMaxSeqs + 2)));
        if (e != cudaSuccess) return fail_cuda("wk_batch_plan", e);
        configured = g_rt.device;
    }
    // one thread per row (or sequence), at most one CTA per SM
    const int work = rows_cap > n ? rows_cap : n;
    int ctas = (work - 1) / kPlanThreads + 1;
    if (ctas > g_rt.num_sms) ctas = g_rt.num_sms;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kPlanThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream();
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = g_rt.pdl ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, batch_plan_kernel, a);
    if (e != cudaSuccess) return fail_cuda("wk_batch_plan", e);
    return 0;
}

}  // extern "C"
