// The description of a step, made on the device from the requests' lengths: where the requests' tokens begin, their
// positions, requests and cache slots, and the block tables, with the pages that requests grow into taken from a list
// of free ones in the requests' order.  With it a step whose lengths only the device knows (how many drafted tokens
// stayed) needs no word from the host.
//
//   q_start[b]  = tokens of the requests before b         kv_len[b] = held[b] + brought[b]
//   pages of b  : ceil(held / page) it has, ceil(kv_len / page) it needs; what it lacks comes from
//                 free_pages[free_start + (pages taken by the requests before b)], and on
//                 (without a list its row holds them already; with have_pages it has as many as that says, where that is
//                 more: those it took for tokens that did not stay)
//   token t of b: position held[b] + (t - q_start[b]), slot page(position / page) * page + position % page
//
// Bound by its launch for a decode step (64 requests of up to 16 pages: 3.3 us) and by the look-ups of the sums and the
// writing of the tables for many requests (250 requests with 47,000 tokens and 2,048 pages each, 3.6 MB: 5.7 us).  One launch and no meeting of CTAs: every CTA adds up all requests by itself (the sums of up to 4,096
// requests are two short scans) and then writes its share of tokens and table words; a new page is worked out again
// by whoever needs it rather than read back from the table.  Rows of `tables` beyond what a request held are written
// by one CTA each and read by none.
#include "common.cuh"
#include "ranges.cuh"

namespace {
constexpr int THREADS = 256;
constexpr int MAX_REQUESTS = 4096;
constexpr int MOST = 0x3fffffff;             // sums stop here instead of running over

struct TableArgs {
    const int* rows;
    const int* held;
    const int* brought;
    int* tables;
    const int* free_pages;
    const int* free_start;
    int* free_next;
    const int* have_pages;                   // null: none behind those that the held tokens lie in
    int* have_next;
    int* q_start;
    int* kv_len;
    int* positions;
    int* seq_of_token;
    int* slots;
    int* block_table;
    int n_requests, n_rows, t_cap, max_pages, page_size;
    int n_free;                              // below zero: no list, the rows hold their pages already
    int* status;
};

__device__ __forceinline__ int add(int a, int b) { return min(a + b, MOST); }

__global__ void __launch_bounds__(THREADS) step_tables_kernel(const TableArgs p) {
    extern __shared__ int shared[];
    int* tok = shared;                       // [n + 1] tokens before each request
    int* fresh = tok + p.n_requests + 1;     // [n + 1] new pages before each request
    int* have = fresh + p.n_requests + 1;    // [n] pages of its row that the step reads from it, or -1: the request is refused
    __shared__ int sums[2][THREADS / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const bool speaks = blockIdx.x == 0;     // one CTA reports and writes what there is one of
    prb_grid_launch_dependents();
    prb_grid_wait();

    // ---- sums over the requests: a run of neighbours a thread, then the warps'
    const int run = (p.n_requests + THREADS - 1) / THREADS;
    const int b0 = min(threadIdx.x * run, p.n_requests), b1 = min(b0 + run, p.n_requests);
    int t_sum = 0, f_sum = 0;
    for (int b = b0; b < b1; ++b) {
        const int row = p.rows[b], held = p.held[b], brought = p.brought[b];
        const int own = p.have_pages != nullptr ? p.have_pages[b] : 0;
        const bool fine = row >= 0 && row < p.n_rows && held >= 0 && brought >= 0 && own >= 0 && own <= p.max_pages &&
                          (long)held + brought <= (long)p.max_pages * p.page_size;
        if (!fine && speaks) {
            if (row < 0 || row >= p.n_rows) prb_set_status(p.status, PRB_S_ROW_RANGE, b, row, p.n_rows);
            else prb_set_status(p.status, PRB_S_POSITION_RANGE, b, held, brought);
        }
        const int w = fine ? (int)(((long)held + brought + p.page_size - 1) / p.page_size) : -1;
        const int h = !fine ? -1 : p.n_free >= 0 ? min(max((int)(((long)held + p.page_size - 1) / p.page_size), own), w) : w;
        have[b] = h;
        tok[b] = t_sum;                      // (within the thread's run, for now)
        fresh[b] = f_sum;
        t_sum = add(t_sum, fine ? brought : 0);
        f_sum = add(f_sum, w - h);
    }
    int t_all = t_sum, f_all = f_sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, t_all, o), f = __shfl_up_sync(0xffffffffu, f_all, o);
        if (lane >= o) {
            t_all = add(t_all, t);
            f_all = add(f_all, f);
        }
    }
    if (lane == 31) {
        sums[0][warp] = t_all;
        sums[1][warp] = f_all;
    }
    __syncthreads();
    int t_before = 0, f_before = 0, t_total = 0, f_total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) {
            t_before = add(t_before, sums[0][w]);
            f_before = add(f_before, sums[1][w]);
        }
        t_total = add(t_total, sums[0][w]);
        f_total = add(f_total, sums[1][w]);
    }
    // (what the lanes before this one hold; a shuffle, since a stopped sum cannot be taken back)
    const int t_up = __shfl_up_sync(0xffffffffu, t_all, 1), f_up = __shfl_up_sync(0xffffffffu, f_all, 1);
    if (lane > 0) {
        t_before = add(t_before, t_up);
        f_before = add(f_before, f_up);
    }
    for (int b = b0; b < b1; ++b) {
        tok[b] = add(tok[b], t_before);
        fresh[b] = add(fresh[b], f_before);
    }
    if (threadIdx.x == 0) {
        tok[p.n_requests] = t_total;
        fresh[p.n_requests] = f_total;
    }
    __syncthreads();
    const int start = p.n_free >= 0 ? *p.free_start : 0;
    auto free_page = [&](int b, int i) -> int {              // the i-th page that b takes
        const long at = (long)start + fresh[b] + i;
        return at >= 0 && at < p.n_free ? p.free_pages[at] : -1;
    };
    if (speaks) {
        for (int b = threadIdx.x; b < p.n_requests; b += THREADS) {
            p.q_start[b] = min(tok[b], p.t_cap);
            p.kv_len[b] = have[b] < 0 ? 0 : p.held[b] + p.brought[b];
            if (p.have_next != nullptr) {
                // pages that it has and those it takes, as far as the list goes; a refused one has what it had
                const long left = start < 0 ? 0 : (long)p.n_free - start - fresh[b];
                const int taken = (int)min(max(left, 0L), (long)(fresh[b + 1] - fresh[b]));
                p.have_next[b] = have[b] < 0 ? p.have_pages[b] : max(p.have_pages[b], have[b] + taken);
            }
        }
        if (threadIdx.x == 0) {
            p.q_start[p.n_requests] = min(t_total, p.t_cap);
            if (t_total > p.t_cap) prb_set_status(p.status, PRB_S_ROW_RANGE, -1, t_total, p.t_cap);
            if (p.n_free >= 0) *p.free_next = add(min(max(start, 0), MOST), f_total);
            if (f_total > 0 && (start < 0 || (long)start + f_total > p.n_free))
                prb_set_status(p.status, PRB_S_PAGE_RANGE, -1, add(min(max(start, -1), MOST), f_total), p.n_free);
        }
    }

    // ---- tokens
    for (int t = blockIdx.x * THREADS + threadIdx.x; t < p.t_cap; t += gridDim.x * THREADS) {
        int pos = 0, req = -1, slot = -1;
        if (t < t_total) {
            int lo = 0, hi = p.n_requests;                    // the last request with tok[b] <= t
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (tok[mid] <= t) lo = mid; else hi = mid;
            }
            req = lo;
            pos = p.held[req] + t - tok[req];
            const int at = pos / p.page_size, in = pos - at * p.page_size;
            const int page = at < have[req] ? p.tables[(size_t)p.rows[req] * p.max_pages + at] : free_page(req, at - have[req]);
            if (page < 0 || page > (0x7fffffff - in) / p.page_size)
                prb_set_status(p.status, PRB_S_PAGE_RANGE, t, pos, page);
            else
                slot = page * p.page_size + in;
        }
        p.positions[t] = pos;
        p.seq_of_token[t] = req;
        p.slots[t] = slot;
    }

    // ---- block tables, a row a CTA at a time
    for (int b = blockIdx.x; b < p.n_requests; b += gridDim.x) {
        const int h = have[b], w = h < 0 ? 0 : h + fresh[b + 1] - fresh[b];
        int* out = p.block_table + (size_t)b * p.max_pages;
        int* table = h < 0 ? nullptr : p.tables + (size_t)p.rows[b] * p.max_pages;
        for (int i = threadIdx.x; i < p.max_pages; i += THREADS) {
            int page = -1;
            if (i < h) {
                page = table[i];
            } else if (i < w) {
                page = free_page(b, i - h);
                table[i] = page;
            }
            out[i] = page;
        }
    }
}
}  // namespace

PRB_API int prb_step_tables(const int* rows, const int* held, const int* brought, int* tables, const int* free_pages,
                            const int* free_start, int* free_next, const int* have_pages, int* have_next, int* q_start,
                            int* kv_len, int* positions, int* seq_of_token, int* slots, int* block_table, int n_requests,
                            int n_rows, int t_cap,
                            int max_pages, int page_size, int n_free, int* status, cudaStream_t stream) {
    if (n_requests <= 0 || n_requests > MAX_REQUESTS || n_rows <= 0 || t_cap < 0 || t_cap > MOST || max_pages <= 0 ||
        page_size <= 0 || (long)max_pages * page_size > 0x7fffffffL)
        return PRB_E_SIZE;
    if (n_free >= 0 && (free_start == nullptr || free_next == nullptr || (n_free > 0 && free_pages == nullptr)))
        return PRB_E_ARG;
    if ((have_pages == nullptr) != (have_next == nullptr) || (have_pages != nullptr && n_free < 0)) return PRB_E_ARG;
    // (a CTA may still read what another writes: the new lengths, for one, must not take the place of those held)
    const long word = sizeof(int), n = n_requests, table = n_rows * (long)max_pages;
    if (!prb_apart({{q_start, (n + 1) * word}, {kv_len, n * word}, {positions, t_cap * word}, {seq_of_token, t_cap * word},
                    {slots, t_cap * word}, {block_table, n * max_pages * word}, {tables, table * word},
                    {n_free >= 0 ? free_next : nullptr, word}, {have_next, n * word}, {status, 4 * word}},
                   {{rows, n * word}, {held, n * word}, {brought, n * word}, {free_pages, n_free * word},
                    {n_free >= 0 ? free_start : nullptr, word}, {have_pages, n * word}}))
        return PRB_E_OVERLAP;
    const TableArgs a{rows, held, brought, tables, free_pages, free_start, free_next, have_pages, have_next, q_start,
                      kv_len, positions, seq_of_token, slots, block_table, n_requests, n_rows, t_cap, max_pages, page_size, n_free, status};
    const int shared = (3 * n_requests + 2) * (int)sizeof(int);
    const cudaError_t a_err = prb_allow_shared<step_tables_kernel>((3 * MAX_REQUESTS + 2) * (int)sizeof(int));
    if (a_err != cudaSuccess) return (int)a_err;
    const long want = max((long)n_requests, ((long)t_cap + THREADS - 1) / THREADS);
    const long most = 4L * prb_sm_count();
    const cudaError_t e = prb_launch_dependent(step_tables_kernel, dim3((unsigned)(want < most ? want : most)),
                                               dim3(THREADS), (size_t)shared, stream, a);
    return e == cudaSuccess ? 0 : (int)e;
}
