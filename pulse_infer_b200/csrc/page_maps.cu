// Block tables and slot maps of a step, built on the GPU from the lengths of its requests.
//
// A step is R segments; segment r brings n = seg_len[r] new tokens of the request in slot seg_slot[r], which already has
// a = seg_start[r] tokens in its pages.  With seg_off the exclusive prefix sum of n:
//   token t of segment r    token_seg[t] = r, positions[t] = p = a + t - seg_off[r],
//                           slot_map[t] = page * page_size + p % page_size with page = block_table[slot, p / page_size]
//                           (64-bit; -1 where the request has no page there)
//   listed pages            a segment of at least min_tokens new tokens lists the pages that its queries can see: with a
//                           window w from page max(0, a - w + 1) / page_size on, otherwise from page 0, to the page of
//                           position a + n - 1.  page_off is the exclusive prefix sum of their counts, page_list the pool
//                           pages one behind the other, page_tokens the tokens [lo, hi) of each that can be seen, and
//                           table[r, i] the place in page_list of the request's page i (-1: not listed).
// (A null table is left out.)  Entries behind the last token or the last listed page are -1 (positions 0, page_tokens empty).
//
// It is latency that counts: a decode step is a few hundred bytes.  So one launch does everything: every block scans the
// R lengths for itself (a few kilobytes out of L2) and then fills its part of the outputs, looking its segment up in the
// sums in shared memory by bisection.
#include "common.cuh"

#define PM_THREADS 256
#define PM_MAX_SEGMENTS 4096
#define PM_PER_BLOCK 2048          // output entries a block fills

struct PmParams {
    const int* block_table; int bt_rows, bt_stride;
    const int* seg_slot; const int* seg_start; const int* seg_len;
    int num_segments, page_shift, num_tokens, num_listed, window, min_tokens;
    long long* slot_map; int* positions; int* token_seg; int* seg_off; int* page_off; int* page_list; int2* page_tokens;
    int* table; int* rows;
};

__device__ __forceinline__ int pm_first_page(const PmParams& p, int start) {
    return p.window > 0 ? max(0, start - p.window + 1) >> p.page_shift : 0;
}

__device__ __forceinline__ int pm_new_tokens(const PmParams& p, int r) { return max(0, p.seg_len[r]); }

__device__ __forceinline__ int pm_listed(const PmParams& p, int start, int n) {
    if (n <= 0 || n < p.min_tokens || start < 0) return 0;
    return ((start + n - 1) >> p.page_shift) - pm_first_page(p, start) + 1;
}

__device__ __forceinline__ int pm_page(const PmParams& p, int r, int index) {
    const int slot = p.seg_slot[r];
    if (slot < 0 || slot >= p.bt_rows || index < 0 || index >= p.bt_stride) return -1;
    return p.block_table[(size_t)slot * p.bt_stride + index];
}

// the segment whose range of an exclusive prefix sum holds i (i is below the total)
__device__ __forceinline__ int pm_owner(const int* sums, int n, int i) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (sums[mid] <= i) lo = mid; else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(PM_THREADS) page_maps_kernel(const PmParams p) {
    extern __shared__ int pm_smem[];                    // [R + 1] token sums, [R + 1] page sums
    __shared__ int warp_tok[PM_THREADS / 32], warp_pg[PM_THREADS / 32];
    int* tok = pm_smem;
    int* pg = pm_smem + p.num_segments + 1;
    const int R = p.num_segments, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // The kernel behind this one is not let in early: the attention kernels look at a step's offsets, slots and lengths before they
    // wait for the kernel in front of them, which is right for what was there before the step, and this kernel writes some of it.
    pdl_wait();
    int base_tok = 0, base_pg = 0;
    for (int first = 0; first < R; first += PM_THREADS) {
        const int r = first + threadIdx.x;
        const int n = r < R ? pm_new_tokens(p, r) : 0;
        const int c = r < R ? pm_listed(p, p.seg_start[r], n) : 0;
        int in = n, ic = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int a = __shfl_up_sync(0xffffffffu, in, o), b = __shfl_up_sync(0xffffffffu, ic, o);
            if (lane >= o) { in += a; ic += b; }
        }
        if (lane == 31) { warp_tok[warp] = in; warp_pg[warp] = ic; }
        __syncthreads();
        int before_tok = base_tok, before_pg = base_pg, all_tok = 0, all_pg = 0;
#pragma unroll
        for (int w = 0; w < PM_THREADS / 32; ++w) {
            if (w < warp) { before_tok += warp_tok[w]; before_pg += warp_pg[w]; }
            all_tok += warp_tok[w]; all_pg += warp_pg[w];
        }
        if (r < R) { tok[r] = before_tok + in - n; pg[r] = before_pg + ic - c; }
        base_tok += all_tok; base_pg += all_pg;
        __syncthreads();
    }
    if (threadIdx.x == 0) { tok[R] = base_tok; pg[R] = base_pg; }
    __syncthreads();

    const int page_size = 1 << p.page_shift;
    const long long cells = p.table != nullptr ? (long long)R * p.bt_stride : 0;
    const long long total = (long long)p.num_tokens + p.num_listed + (R + 1) + cells;
    const long long begin = (long long)blockIdx.x * PM_PER_BLOCK;
    const long long end = min(begin + PM_PER_BLOCK, total);
    for (long long u = begin + threadIdx.x; u < end; u += PM_THREADS) {
        long long i = u;
        if (i < p.num_tokens) {
            const int t = (int)i;
            int seg = -1, pos = 0;
            long long slot = -1;
            if (t < base_tok) {
                seg = pm_owner(tok, R, t);
                pos = p.seg_start[seg] + t - tok[seg];
                const int page = pos >= 0 ? pm_page(p, seg, pos >> p.page_shift) : -1;
                if (page >= 0) slot = ((long long)page << p.page_shift) + (pos & (page_size - 1));
            }
            p.slot_map[t] = slot; p.positions[t] = pos; p.token_seg[t] = seg;
            continue;
        }
        i -= p.num_tokens;
        if (i < p.num_listed) {
            const int k = (int)i;
            int page = -1;
            int2 span = make_int2(0, 0);
            if (k < base_pg) {
                const int seg = pm_owner(pg, R, k);
                const int start = p.seg_start[seg], index = pm_first_page(p, start) + k - pg[seg];
                const int lo = p.window > 0 ? max(0, start - p.window + 1) : 0, hi = start + pm_new_tokens(p, seg);
                page = pm_page(p, seg, index);
                span = make_int2(max(0, lo - (index << p.page_shift)), min(page_size, hi - (index << p.page_shift)));
            }
            p.page_list[k] = page; p.page_tokens[k] = span;
            continue;
        }
        i -= p.num_listed;
        if (i <= R) {
            p.seg_off[i] = tok[i]; p.page_off[i] = pg[i];
            if (i < R) p.rows[i] = (int)i;
            continue;
        }
        i -= R + 1;
        const int r = (int)(i / p.bt_stride), index = (int)(i - (long long)r * p.bt_stride);
        const int place = index - pm_first_page(p, p.seg_start[r]), count = pg[r + 1] - pg[r];
        p.table[i] = (place >= 0 && place < count && pg[r] + place < p.num_listed) ? pg[r] + place : -1;
    }
}

// arguments as one record of 8-byte fields (one pointer to pass instead of 22 values)
struct PmArgs {
    const int* block_table; long long bt_rows, bt_stride;
    const int* seg_slot; const int* seg_start; const int* seg_len;
    long long num_segments, page_size, num_tokens, num_listed, window, min_tokens;
    long long* slot_map; int* positions; int* token_seg; int* seg_off; int* page_off; int* page_list; int* page_tokens;
    int* table; int* rows;
};

PI_EXPORT int pi_page_maps(const PmArgs* args, cudaStream_t stream) {
    const PmArgs& a = *args;
    const int bt_rows = (int)a.bt_rows, bt_stride = (int)a.bt_stride, num_segments = (int)a.num_segments, page_size = (int)a.page_size;
    const int num_tokens = (int)a.num_tokens, num_listed = (int)a.num_listed, window = (int)a.window, min_tokens = (int)a.min_tokens;
    if (num_segments <= 0) return pi_refuse("pi_page_maps: num_segments=%d must be positive", num_segments);
    if (num_segments > PM_MAX_SEGMENTS) return pi_refuse("pi_page_maps: %d segments; at most %d", num_segments, PM_MAX_SEGMENTS);
    if (page_size <= 0 || (page_size & (page_size - 1))) return pi_refuse("pi_page_maps: page_size=%d must be a power of two", page_size);
    if (num_tokens < 0 || num_listed < 0 || window < 0 || min_tokens < 1 || bt_rows <= 0 || bt_stride <= 0)
        return pi_refuse("pi_page_maps: num_tokens=%d num_listed=%d window=%d min_tokens=%d table [%d, %d]", num_tokens, num_listed,
                         window, min_tokens, bt_rows, bt_stride);
    PmParams p;
    p.block_table = a.block_table; p.bt_rows = bt_rows; p.bt_stride = bt_stride;
    p.seg_slot = a.seg_slot; p.seg_start = a.seg_start; p.seg_len = a.seg_len;
    p.num_segments = num_segments; p.num_tokens = num_tokens; p.num_listed = num_listed; p.window = window; p.min_tokens = min_tokens;
    p.page_shift = 0;
    while ((1 << p.page_shift) < page_size) ++p.page_shift;
    p.slot_map = a.slot_map; p.positions = a.positions; p.token_seg = a.token_seg; p.seg_off = a.seg_off; p.page_off = a.page_off;
    p.page_list = a.page_list; p.page_tokens = (int2*)a.page_tokens; p.table = a.table; p.rows = a.rows;
    const long long total = (long long)num_tokens + num_listed + num_segments + 1 + (a.table != nullptr ? (long long)num_segments * bt_stride : 0);
    const long long blocks = (total + PM_PER_BLOCK - 1) / PM_PER_BLOCK;
    if (blocks > 2147483647LL) return pi_refuse("pi_page_maps: %lld entries are beyond the grid limit", total);
    const size_t smem = 2 * (size_t)(num_segments + 1) * sizeof(int);       // at most 32 KB: within the default limit
    pi_launch(page_maps_kernel, dim3((unsigned)blocks), dim3(PM_THREADS), smem, stream, p);
    return pi_check_launch("pi_page_maps");
}
