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

constexpr int kPlanThreads = 256;
constexpr int kPlanRows = 2048;          // rows of the step per CTA of the cluster, up to eight CTAs
constexpr int kPlanMaxB = 16384;         // three words of shared memory per request
constexpr int kNoRoom = INT32_MIN, kNoPages = INT32_MIN + 1;      // in place of a stack index, which is above -2^30

// exclusive sum over the block's threads; `total` for all of them. Two barriers; `part` may be used again behind the second.
template <typename T>
__device__ __forceinline__ T block_scan(T v, T* part, T& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    T in = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T u = __shfl_up_sync(0xFFFFFFFFu, in, o);
        if (lane >= o) in += u;
    }
    if (lane == 31) part[warp] = in;
    __syncthreads();
    T before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 32; ++w) {
        const T s = part[w];
        if (w < warp) before += s;
        total += s;
    }
    __syncthreads();
    return before + in - v;
}

__device__ __forceinline__ int pages_of(int tokens, int page) { return (int)(((unsigned)tokens + (unsigned)page - 1u) / (unsigned)page); }

__global__ void __launch_bounds__(kPlanThreads)
page_plan_kernel(const PagePlanArgs a) {
    extern __shared__ int sm[];
    __shared__ long long part64[kPlanThreads / 32];
    __shared__ int part32[kPlanThreads / 32];
    int *start = sm, *base = start + a.B + 1, *have = base + a.B;      // first row, stack index of page 0 (page j is below it by j), cached tokens
    const int tid = threadIdx.x, cta = blockIdx.x, ctas = gridDim.x;
    const int per = (a.B + kPlanThreads - 1) / kPlanThreads, b0 = min(a.B, tid * per), b1 = min(a.B, b0 + per);
    const long long room = min((long long)a.width * a.page_size, (long long)INT32_MAX);
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
    long long row = block_scan(rows, part64, all_rows);
    int need = 0, back = 0, all_need, all_back;
    for (int b = b0; b < b1; ++b) {
        const int n = base[b], c = have[b], add = max(n, 0);
        const long long first = a.row_pitch > 0 ? (long long)b * a.row_pitch : row;
        start[b] = (int)min(first, (long long)INT32_MAX);
        row += add;
        if (c < 0 || c + (long long)add > room || (add > 0 && (first + add > a.max_rows || (a.row_pitch > 0 && add > a.row_pitch)))) base[b] = kNoRoom;
        else if (n < 0) back += pages_of(c, a.page_size);
        else need += pages_of(c + n, a.page_size) - pages_of(c, a.page_size);
    }
    if (tid == 0) start[a.B] = (int)min(a.row_pitch > 0 ? (long long)a.B * a.row_pitch : all_rows, (long long)INT32_MAX);
    int before = block_scan(need, part32, all_need), put = block_scan(back, part32, all_back), taken = 0;
    // served are the requests that need nothing and the leading ones of the others: what is taken is the largest sum within the free pages
    for (int b = b0; b < b1; ++b) {
        const int n = base[b], c = have[b];
        if (n == kNoRoom) continue;
        const int held = pages_of(c, a.page_size);
        if (n < 0) { base[b] = put; put += held; continue; }
        const int want = pages_of(c + n, a.page_size) - held;
        before += want;
        const bool served = want == 0 || before <= n_free;
        base[b] = served ? n_free - 1 - (before - want) + held : kNoPages;
        if (served && want) taken = before;
    }
    taken = __reduce_max_sync(0xFFFFFFFFu, taken);
    if ((tid & 31) == 0) part32[tid >> 5] = taken;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kPlanThreads / 32; ++w) taken = max(taken, part32[w]);

    for (int r = cta * kPlanThreads + tid; r < a.max_rows; r += ctas * kPlanThreads) {
        int b;
        if (a.row_pitch > 0) {
            b = min(r / a.row_pitch, a.B);
        } else {
            int lo = 0, hi = a.B + 1;            // the last b with start[b] <= r: of several that start here the one that has rows
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (start[mid] <= r) lo = mid; else hi = mid;
            }
            b = lo;
        }
        int slot = -1, pos = -1;
        if (b < a.B && base[b] > kNoPages) {
            const int t = r - start[b], c = have[b];
            if (t < a.new_tokens[b]) {
                pos = c + t;
                const int j = pos / a.page_size, in = pos - j * a.page_size;
                int* entry = a.table + (long long)b * a.ldt + j;
                int id;
                if (j < pages_of(c, a.page_size)) {
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
    if (ctas > 1) cluster_sync_all(); else __syncthreads();      // lengths may be cached, and what is given back goes where pages were taken from
    if (cta != 0) return;
    const int left = n_free - taken;
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
        const int held = pages_of(have[b], a.page_size), at = left + base[b];
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

// A row per blockDim.x threads and step; UN steps of a thread are requested together.
template <int UN>
__global__ void __launch_bounds__(256)
page_write_kernel(const PageWriteParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const int step = gridDim.x * blockDim.y;
    for (int r0 = blockIdx.x * blockDim.y + threadIdx.y; r0 < p.rows; r0 += step * UN) {
        int slot[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) slot[u] = r0 + u * step < p.rows ? p.slots[r0 + u * step] : -1;
        for (int c = threadIdx.x; c < p.vecs; c += blockDim.x) {
            uint4 k[UN], v[UN];
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                if ((unsigned)slot[u] >= (unsigned)p.n_slots) continue;
                k[u] = __ldcs(p.k + (r0 + u * step) * p.ldk + c);
                v[u] = __ldcs(p.v + (r0 + u * step) * p.ldv + c);
            }
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                if ((unsigned)slot[u] >= (unsigned)p.n_slots) continue;
                const int pg = slot[u] / p.page;
                const long long at = pg * p.page_stride + (slot[u] - pg * p.page) * p.tok_stride + c;
                p.kp[at] = k[u];
                p.vp[at] = v[u];
            }
        }
    }
}

}  // namespace

int launch_page_plan(const PagePlanArgs& a, cudaStream_t stream) {
    if (a.B > kPlanMaxB) { set_last_error("page_plan: %d requests exceed %d", a.B, kPlanMaxB); return PLZ_ERR_TOO_LARGE; }
    const size_t smem = (size_t)(3 * a.B + 1) * sizeof(int);
    if (smem > 40 * 1024) PLZ_CUDA_CHECK(cudaFuncSetAttribute(page_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (kPlanMaxB * 3 + 1) * (int)sizeof(int)));
    int ctas = 1;
    while (ctas < 8 && ctas * kPlanRows < a.max_rows) ctas *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas); cfg.blockDim = dim3(kPlanThreads); cfg.dynamicSmemBytes = smem; cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr; cfg.numAttrs = behind_attr(stream, attr);
    if (g_smallm_overlap) cfg.numAttrs = 1;
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = ctas; attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
    PLZ_CUDA_CHECK(cudaLaunchKernelEx(&cfg, page_plan_kernel, a));
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
    const int sms = sms_of_current_device(), groups = (a.rows + (int)block.y - 1) / (int)block.y;
    if (groups <= 8 * sms) PLZ_LAUNCH_CHAIN_BEHIND(page_write_kernel<1>, dim3(groups), block, 0, stream, p);
    else PLZ_LAUNCH_CHAIN_BEHIND(page_write_kernel<4>, dim3(8 * sms < (groups + 3) / 4 ? 8 * sms : (groups + 3) / 4), block, 0, stream, p);
    return PLZ_OK;
}

}  // namespace plz
