// Pages of a key / value cache for a batch of requests of different lengths: which pages and slots a step's new tokens get, and the write of their keys and values.
//
//   page_plan_kernel  Request b holds held = ceil(cached / page) pages and brings n tokens: it needs ceil((cached + n) / page) - held more. Requests are served in
//     order while the running sum of what they need is covered by the free pages; page j of a request (j >= held) is free[n_free - 1 - (sum before b) - (j - held)],
//     so what a request gets follows from two prefix sums, and every row (new token) finds its request by a search in the starts and computes its slot alone.
//     One cluster: every CTA makes both sums for itself (B numbers, a few hundred), takes its share of the rows, and the lengths and the count of free pages, which may be
//     the inputs themselves, are written behind a barrier that all have passed.
//   page_write_kernel  row i of k and v to slot slots[i]; bound by memory: every byte is read once and written once, 16 bytes a thread and access.
#include "plz_launch.h"

namespace plz {
namespace {

constexpr int kPlanRows = 1024;          // rows of the step per CTA of the cluster, up to eight CTAs
constexpr int kPlanMaxB = 16384;         // three words of shared memory per request
constexpr int kNoRoom = INT32_MIN, kNoPages = INT32_MIN + 1;      // in place of a stack index, which is above -2^30

// exclusive sum over the block's threads, `total` for all of them; `part` may be used again behind another barrier
template <int kPlanThreads>
__device__ __forceinline__ long long block_scan(long long v, long long* part, long long& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long in = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xFFFFFFFFu, in, o);
        if (lane >= o) in += u;
    }
    if (lane == 31) part[warp] = in;
    __syncthreads();
    long long all = lane < kPlanThreads / 32 ? part[lane] : 0;            // every warp sums up the warps for itself
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xFFFFFFFFu, all, o);
        if (lane >= o) all += u;
    }
    total = __shfl_sync(0xFFFFFFFFu, all, 31);
    return in - v + (warp ? __shfl_sync(0xFFFFFFFFu, all, warp - 1) : 0);
}

struct Pages {                             // divisions by the page size
    int size, shift;
    __device__ __forceinline__ int of(int tokens) const { return shift >= 0 ? (int)(((unsigned)tokens + (unsigned)size - 1u) >> shift) : (int)(((unsigned)tokens + (unsigned)size - 1u) / (unsigned)size); }
    __device__ __forceinline__ int at(int pos) const { return shift >= 0 ? pos >> shift : pos / size; }
};

template <int kPlanThreads, int kPlanRowsAtOnce>
__global__ void __launch_bounds__(kPlanThreads, 1)
page_plan_kernel(const PagePlanArgs a) {
    extern __shared__ int sm[];
    __shared__ long long part[2][kPlanThreads / 32];
    __shared__ int sm_taken;
    int *start = sm, *base = start + a.B + 1, *have = base + a.B;      // first row, stack index of page 0 (page j is below it by j), cached tokens
    const int tid = threadIdx.x, cta = blockIdx.x, ctas = gridDim.x;
    const int per = (a.B + kPlanThreads - 1) / kPlanThreads, b0 = min(a.B, tid * per), b1 = min(a.B, b0 + per);
    const long long room = min((long long)a.width * a.page_size, (long long)(a.max_tokens ? a.max_tokens : INT32_MAX));
    const Pages pages = {a.page_size, (a.page_size & (a.page_size - 1)) == 0 ? __ffs(a.page_size) - 1 : -1};
    if (tid == 0) sm_taken = 0;
    pdl_launch_dependents();
    pdl_wait();
    const int n_free = min(max(*a.n_free, 0), a.n_pages);

    long long rows = 0, all_rows;
    for (int b = b0; b < b1; ++b) {
        const int n = a.new_tokens[b];
        have[b] = a.cached[b];
        base[b] = n;
        rows += max(n, 0);
    }
    long long row = block_scan<kPlanThreads>(rows, part[0], all_rows);
    unsigned need = 0, back = 0;           // each below 2^30 in all
    for (int b = b0; b < b1; ++b) {
        const int n = base[b], c = have[b], add = max(n, 0);
        const long long first = a.row_pitch > 0 ? (long long)b * a.row_pitch : row;
        start[b] = (int)min(first, (long long)INT32_MAX);
        row += add;
        if (c < 0 || c + (long long)add > room || (add > 0 && (first + add > a.max_rows || (a.row_pitch > 0 && add > a.row_pitch)))) base[b] = kNoRoom;
        else if (n < 0) back += pages.of(c);
        else need += pages.of(c + n) - pages.of(c);
    }
    if (tid == 0) start[a.B] = (int)min(a.row_pitch > 0 ? (long long)a.B * a.row_pitch : all_rows, (long long)INT32_MAX);
    long long both;
    const long long ahead = block_scan<kPlanThreads>((long long)back << 32 | need, part[1], both);
    int before = (int)(unsigned)ahead, put = (int)(ahead >> 32), taken = 0;
    const int all_back = (int)(both >> 32);
    // served are the requests that need nothing and the leading ones of the others: what is taken is the largest sum within the free pages
    for (int b = b0; b < b1; ++b) {
        const int n = base[b], c = have[b];
        if (n == kNoRoom) continue;
        const int held = pages.of(c);
        if (n < 0) { base[b] = put; put += held; continue; }
        const int want = pages.of(c + n) - held;
        before += want;
        const bool served = want == 0 || before <= n_free;
        base[b] = served ? n_free - 1 - (before - want) + held : kNoPages;
        if (served && want) taken = before;
    }
    if (cta == 0) {                        // nobody else needs it
        taken = __reduce_max_sync(0xFFFFFFFFu, taken);
        if ((tid & 31) == 0 && taken) atomicMax(&sm_taken, taken);
    }
    __syncthreads();

    // rows, kPlanRowsAtOnce of a thread side by side: a search is a chain of shared-memory reads. Bound by issue on the cluster's few SMs (32768 rows of 1000 requests 8.2 us, 9.9 with a branch in the search).
    for (int r0 = cta * kPlanThreads + tid; r0 < a.max_rows; r0 += ctas * kPlanThreads * kPlanRowsAtOnce) {
        int lo[kPlanRowsAtOnce], hi[kPlanRowsAtOnce];
#pragma unroll
        for (int u = 0; u < kPlanRowsAtOnce; ++u) { lo[u] = 0; hi[u] = a.B + 1; }
        if (a.row_pitch > 0) {
#pragma unroll
            for (int u = 0; u < kPlanRowsAtOnce; ++u) lo[u] = min((r0 + u * ctas * kPlanThreads) / a.row_pitch, a.B);
        } else {
            // the last b with start[b] <= r: of several that start here the one that has rows. All searches take the same number of turns.
            for (int left = a.B; left > 0; left >>= 1)
#pragma unroll
                for (int u = 0; u < kPlanRowsAtOnce; ++u) {
                    const int mid = (lo[u] + hi[u]) >> 1;      // lo itself once nothing lies between, whose start is not behind r
                    const bool up = start[mid] <= r0 + u * ctas * kPlanThreads;
                    lo[u] = up ? mid : lo[u];
                    hi[u] = up ? hi[u] : mid;
                }
        }
#pragma unroll
        for (int u = 0; u < kPlanRowsAtOnce; ++u) {
            const int r = r0 + u * ctas * kPlanThreads, b = lo[u];
            if (r >= a.max_rows) break;
            int slot = -1, pos = -1;
            if (b < a.B && base[b] > kNoPages) {
                const int t = r - start[b], c = have[b];
                if (a.row_pitch == 0 || t < a.new_tokens[b]) {
                    pos = c + t;
                    const int j = pages.at(pos), in = pos - j * a.page_size;
                    int* entry = a.table + (long long)b * a.ldt + j;
                    int id;
                    if (j < pages.of(c)) {
                        id = *entry;
                    } else {
                        id = a.free_pages[base[b] - j];
                        if (in == 0) *entry = id;
                    }
                    slot = (unsigned)id < (unsigned)a.n_pages ? id * a.page_size + in : -1;
                }
            }
            a.slots[r] = slot;
            a.positions[r] = pos;
        }
    }
    if (ctas > 1) cluster_sync_all(); else __syncthreads();      // lengths may be cached, and what is given back goes where pages were taken from
    if (cta != 0) return;
    const int left = n_free - sm_taken;
    for (int b = b0; b < b1; ++b) {
        const int n = a.new_tokens[b], c = have[b], at = base[b];
        a.lengths[b] = at <= kNoPages ? c : n < 0 ? 0 : c + n;
        a.status[b] = at == kNoRoom ? 2 : at == kNoPages ? 1 : 0;
        a.starts[b] = start[b];
    }
    if (tid == 0) {
        a.starts[a.B] = start[a.B];
        *a.n_free_out = min(left + all_back, a.n_pages);
    }
    if (all_back == 0) return;
    for (int b = tid >> 5; b < a.B; b += kPlanThreads / 32) {
        if (base[b] <= kNoPages || a.new_tokens[b] >= 0) continue;
        const int held = pages.of(have[b]), at = left + base[b];
        for (int j = tid & 31; j < held; j += 32)
            if (at + j < a.n_pages) a.free_pages[at + j] = a.table[(long long)b * a.ldt + j];
    }
}

struct PageWriteParams {
    const uint4 *k, *v; long long ldk, ldv;             // 16-byte units between rows
    uint4 *kp, *vp; long long page_stride, tok_stride;  // 16-byte units
    const int* slots;
    int rows, vecs, page, n_slots;
};

// A row per blockDim.x threads, a 16-byte unit of k and of v a thread. More rows of a thread at once, or fewer CTAs that loop, are slower: 16383 rows of 2 KB 21.7 us, two rows 21.7, four 22.3,
// eight 24.5 us. PASS: more than L2 keeps until it is read; streaming stores then 20.7 us.
template <bool PASS>
__global__ void __launch_bounds__(256)
page_write_kernel(const PageWriteParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const int r = blockIdx.x * blockDim.y + threadIdx.y;
    if (r >= p.rows) return;
    const int slot = p.slots[r];
    if ((unsigned)slot >= (unsigned)p.n_slots) return;
    const int pg = slot / p.page;
    const long long to = pg * p.page_stride + (slot - pg * p.page) * p.tok_stride;
    for (int c = threadIdx.x; c < p.vecs; c += blockDim.x) {
        const uint4 k = __ldcs(p.k + r * p.ldk + c), v = __ldcs(p.v + r * p.ldv + c);
        if (PASS) {
            __stcs(p.kp + to + c, k);
            __stcs(p.vp + to + c, v);
        } else {
            p.kp[to + c] = k;
            p.vp[to + c] = v;
        }
    }
}

}  // namespace

int launch_page_plan(const PagePlanArgs& a, cudaStream_t stream) {
    if (a.B > kPlanMaxB) { set_last_error("page_plan: %d requests exceed %d", a.B, kPlanMaxB); return PLZ_ERR_TOO_LARGE; }
    // few requests and rows: a small CTA, without the cluster's launch (64 requests with a row each 5.4 -> 3.3 us)
    if (a.B <= 256 && a.max_rows <= 256) {
        PLZ_LAUNCH_CHAIN_BEHIND((page_plan_kernel<256, 1>), dim3(1), dim3(256), (size_t)(3 * a.B + 1) * sizeof(int), stream, a);
        return PLZ_OK;
    }
    auto kern = page_plan_kernel<1024, 4>;
    const size_t smem = (size_t)(3 * a.B + 1) * sizeof(int);
    if (smem > 40 * 1024) PLZ_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (kPlanMaxB * 3 + 1) * (int)sizeof(int)));
    int ctas = 1;
    while (ctas < 8 && ctas * kPlanRows < a.max_rows) ctas *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas); cfg.blockDim = dim3(1024); cfg.dynamicSmemBytes = smem; cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr; cfg.numAttrs = behind_attr(stream, attr);
    if (g_smallm_overlap) cfg.numAttrs = 1;
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = ctas; attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
    PLZ_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, a));
    ++g_launch_count;
    return PLZ_OK;
}

int launch_page_write(const PageWriteArgs& a, cudaStream_t stream) {
    if (a.rows <= 0) return PLZ_OK;
    const PageWriteParams p = {(const uint4*)a.k, (const uint4*)a.v, a.ldk / 16, a.ldv / 16, (uint4*)a.k_pages, (uint4*)a.v_pages, a.page_stride / 16, a.tok_stride / 16,
                               a.slots, a.rows, a.row_bytes / 16, a.page_size, (int)((long long)a.n_pages * a.page_size)};
    int tx = 8;
    while (tx < 256 && tx < p.vecs) tx *= 2;
    const dim3 block(tx, 256 / tx);
    const dim3 grid((unsigned)((a.rows + (int)block.y - 1) / (int)block.y));
    if ((long long)a.rows * a.row_bytes > (16 << 20)) PLZ_LAUNCH_CHAIN_BEHIND(page_write_kernel<true>, grid, block, 0, stream, p);
    else PLZ_LAUNCH_CHAIN_BEHIND(page_write_kernel<false>, grid, block, 0, stream, p);
    return PLZ_OK;
}

}  // namespace plz
