// What a request's settings do to its logits before a token is picked: penalties for tokens that occurred, biases of single tokens, a grammar's mask.
//
//   x = x > 0 ? x / r : x * r  for tokens that occur;  x - f * c - p  for those that occur c > 0 times behind the prompt;  + biases;  -inf where the mask has a 0.
//
// Bound by memory (a logit read and written once) from a few rows on. Few tokens of a vocabulary are touched, so the penalties and biases stay out of the stream of all logits: with them in it,
// 50 instructions a logit, 64 rows of 151936 took 30 us, bound by issue.
//   A CTA takes a segment of a row, copies it through the mask, 16 bytes a thread and access, and counts the row's tokens that fall into it in shared memory (whole numbers, exact in any order);
//   reading all tokens in every CTA costs less than a cluster that reads them once and counts in its distributed shared memory (8 rows with 30000 tokens 18 us, 64 rows 38 us: its CTAs wait for one
//   another, and its atomics are slow). One warp lists the biases of the segment's tokens in their order and marks the tokens' counts; several biases of one token are added in the order of
//   the row's list whatever the threads do. Then the tokens with a mark are listed, their logits computed by all threads alike and stored over the copy.
#include "plz_launch.h"

namespace plz {
namespace {

constexpr int kAdjFirst = 2, kAdjUnits = 4, kAdjTokens = 8;      // 16-byte units (first ones, later ones) and tokens of a thread that are on their way at once
// logits of a CTA of 512 threads (counts of 16 bits, histories of up to 8192 tokens) and of 1024 (of 32 bits) at most: what shared memory holds of counts, list and biases
constexpr int kAdjLargest = 40960, kAdjLargestLong = 32768, kAdjShort = 8192;
constexpr int kAdjBiases = 4096;         // of a row at most

// a token's mark: occurs, has a bias, how often behind the prompt
template <bool SHORT> struct Mark;
template <> struct Mark<false> { static constexpr uint32_t kSeen = 0x80000000u, kBiased = 0x40000000u, kCount = 0x3FFFFFFFu; };
template <> struct Mark<true> { static constexpr uint32_t kSeen = 0x8000u, kBiased = 0x4000u, kCount = 0x3FFFu; };

struct AdjParams {
    const void* in; long long ld;
    void* out; long long ldo;
    const long long* tokens; long long ldk;
    const int *lengths, *prompt_lengths;
    const float *repetition, *presence, *frequency;
    const long long* bias_ids; const float* bias; long long ldb;
    const int* mask; long long ldm;
    float repetition_all, presence_all, frequency_all;
    int V, max_tokens, n_bias, seg;
};

template <typename T> struct Pack;
template <> struct Pack<float> {
    static constexpr int N = 4;
    __device__ __forceinline__ static float get(float v) { return v; }
    __device__ __forceinline__ static float put(float v) { return v; }
    // -inf where the bit is 0
    __device__ __forceinline__ static uint4 masked(const uint4& v, uint32_t bits) {
        return make_uint4(bits & 1u ? v.x : 0xFF800000u, bits & 2u ? v.y : 0xFF800000u, bits & 4u ? v.z : 0xFF800000u, bits & 8u ? v.w : 0xFF800000u);
    }
};
template <> struct Pack<__nv_bfloat16> {
    static constexpr int N = 8;
    __device__ __forceinline__ static float get(__nv_bfloat16 v) { return __bfloat162float(v); }
    __device__ __forceinline__ static __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
    __device__ __forceinline__ static uint32_t two(uint32_t w, uint32_t bits) { return (bits & 1u ? w & 0xFFFFu : 0xFF80u) | (bits & 2u ? w & 0xFFFF0000u : 0xFF800000u); }
    __device__ __forceinline__ static uint4 masked(const uint4& v, uint32_t bits) { return make_uint4(two(v.x, bits), two(v.y, bits >> 2), two(v.z, bits >> 4), two(v.w, bits >> 6)); }
};

struct RowSettings { float r, p, f; };

template <typename M>
__device__ __forceinline__ float penalized(float x, uint32_t n, const RowSettings& s) {
    const uint32_t c = n & M::kCount;
    if (n & (M::kSeen | M::kCount)) x = x > 0.f ? x / s.r : x * s.r;
    return c ? x - s.f * (float)c - s.p : x;
}

// CTA c has the `seg` logits from c * seg behind the row's first 16-byte boundary on, the first CTA the few in front of it too. A CTA's logits have numbers of their own, `own`: logit t
// is N + t - v0, so that a unit's counts begin on a 16-byte boundary.
template <typename T, int kAdjThreads>
__global__ void __launch_bounds__(kAdjThreads, 1024 / kAdjThreads)
adjust_logits_kernel(const AdjParams p) {
    constexpr int N = Pack<T>::N;
    constexpr bool SHORT = kAdjThreads == 512;
    constexpr int PER = SHORT ? 8 : 4;                                      // counts in 16 bytes
    typedef Mark<SHORT> M;
    extern __shared__ __align__(16) uint32_t count[];                       // N + seg counts, of 16 bits two a word
    const int words16 = (N + p.seg + PER - 1) / PER;                        // 16-byte words of them
    auto mark = [&](int own, uint32_t what, bool add) {
        uint32_t* const where = SHORT ? count + own / 2 : count + own;
        if (SHORT) what <<= (own & 1) * 16;
        if (add) atomicAdd(where, what); else atomicOr(where, what);
    };
    auto marked = [&](int own) { return SHORT ? (uint32_t)reinterpret_cast<const uint16_t*>(count)[own] : count[own]; };
    __shared__ int sm_list, sm_biases;
    int* const ids = reinterpret_cast<int*>(count + words16 * 4);           // biases of this CTA's tokens
    float* const bias = reinterpret_cast<float*>(ids + p.n_bias);
    uint16_t* const list = reinterpret_cast<uint16_t*>(bias + p.n_bias);   // own numbers of the tokens with a mark
    const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
    const T* in = (const T*)p.in + row * p.ld;
    T* out = (T*)p.out + row * p.ldo;
    const int head = min((int)(((16u - (uint32_t)((uintptr_t)in & 15)) & 15u) / sizeof(T)), p.V);
    const int v0 = min(head + (int)blockIdx.x * p.seg, p.V), s0 = blockIdx.x ? v0 : 0, s1 = blockIdx.x + 1 == gridDim.x ? p.V : min(v0 + p.seg, p.V);
    const bool vec = (((uintptr_t)(out + head)) & 15) == 0, marks = (p.lengths && p.max_tokens > 0) || p.n_bias > 0;
    if (marks) {
        for (int i = tid; i < words16; i += kAdjThreads) reinterpret_cast<uint4*>(count)[i] = make_uint4(0u, 0u, 0u, 0u);
        if (tid == 0) sm_list = sm_biases = 0;
    }
    pdl_launch_dependents();
    pdl_wait();
    const int* mask = p.mask ? p.mask + row * p.ldm : nullptr;
    const int words = (p.V + 31) >> 5;
    // a unit of 16 bytes and its mask words, shifted when they are needed
    struct Unit { uint4 raw; uint32_t lo, hi; };
    auto load = [&](int t, Unit& u) {
        u.lo = u.hi = 0xFFFFFFFFu;
        if (!vec || t + N > s1) return;
        u.raw = *reinterpret_cast<const uint4*>(in + t);
        if (mask) {
            const int w = t >> 5;
            u.lo = mask[w];
            u.hi = mask[min(w + 1, words - 1)];
        }
    };
    Unit first[kAdjFirst];                     // on their way while tokens are counted
#pragma unroll
    for (int k = 0; k < kAdjFirst; ++k) load(v0 + (k * kAdjThreads + tid) * N, first[k]);
    if (marks) {
        // the first tokens are asked for ahead of knowing how many there are
        const int most = p.lengths ? p.max_tokens : 0;
        const long long* tok = p.tokens + row * p.ldk;
        constexpr int U = kAdjTokens;          // tokens of a thread that are asked for together
        long long t[U];
        auto fetch = [&](int i0) {
#pragma unroll
            for (int u = 0; u < U; ++u) t[u] = i0 + u * kAdjThreads < most ? tok[i0 + u * kAdjThreads] : -1;
        };
        int i0 = tid;
        fetch(i0);
        constexpr int UB = 4;
        const bool lists = p.n_bias > 0 && tid >= kAdjThreads - 32;
        long long id[UB];
        float v[UB];
        auto fetch_biases = [&](int j0) {
#pragma unroll
            for (int u = 0; u < UB; ++u) {
                const bool more = j0 + 32 * u < p.n_bias;
                id[u] = more ? p.bias_ids[row * p.ldb + j0 + 32 * u] : -1;
                v[u] = more ? p.bias[row * p.ldb + j0 + 32 * u] : 0.f;
            }
        };
        if (lists) fetch_biases(lane);
        const int n_tok = p.lengths ? min(max(p.lengths[row], 0), p.max_tokens) : 0, n_prompt = p.prompt_lengths ? max(p.prompt_lengths[row], 0) : 0;
        __syncthreads();                       // all counts are 0
        if (lists) {
            // one warp keeps what belongs to this CTA, in its order
            int n = 0;
            for (int j0 = lane; j0 - lane < p.n_bias; j0 += 32 * UB) {
#pragma unroll
                for (int u = 0; u < UB; ++u) {
                    const bool mine = id[u] >= s0 && id[u] < s1;
                    const int own = N + (int)id[u] - v0;
                    const uint32_t all = __ballot_sync(0xFFFFFFFFu, mine);
                    if (mine) {
                        const int at = n + __popc(all & ((1u << lane) - 1u));
                        ids[at] = own;
                        bias[at] = v[u];
                        mark(own, M::kBiased, false);
                    }
                    n += __popc(all);
                }
                fetch_biases(j0 + 32 * UB);
            }
            if (lane == 0) sm_biases = n;
        }
        for (; i0 < n_tok; i0 += kAdjThreads * U) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (t[u] < s0 || t[u] >= s1 || i0 + u * kAdjThreads >= n_tok) continue;
                const bool own_word = i0 + u * kAdjThreads >= n_prompt;
                mark(N + (int)t[u] - v0, own_word ? 1u : M::kSeen, own_word);
            }
            fetch(i0 + kAdjThreads * U);
        }
    }
    // all logits
    auto store = [&](int t, Unit& u) {
        if (t >= s1) return;
        if (vec && t + N <= s1) {
            if (mask) u.raw = Pack<T>::masked(u.raw, __funnelshift_r(u.lo, u.hi, t & 31));
            *reinterpret_cast<uint4*>(out + t) = u.raw;
        } else {
            // the row's end, or in and out lie differently
            for (int e = 0; e < N && t + e < s1; ++e) out[t + e] = !mask || ((mask[(t + e) >> 5] >> ((t + e) & 31)) & 1) ? in[t + e] : Pack<T>::put(-INFINITY);
        }
    };
#pragma unroll
    for (int k = 0; k < kAdjFirst; ++k) store(v0 + (k * kAdjThreads + tid) * N, first[k]);
    for (int t0 = v0 + kAdjFirst * kAdjThreads * N; t0 < s1; t0 += kAdjUnits * kAdjThreads * N) {
        Unit unit[kAdjUnits];
#pragma unroll
        for (int k = 0; k < kAdjUnits; ++k) load(t0 + (k * kAdjThreads + tid) * N, unit[k]);
#pragma unroll
        for (int k = 0; k < kAdjUnits; ++k) store(t0 + (k * kAdjThreads + tid) * N, unit[k]);
    }
    if (tid < v0 - s0) out[tid] = !mask || ((mask[0] >> tid) & 1) ? in[tid] : Pack<T>::put(-INFINITY);
    if (!marks) return;
    RowSettings s;
    s.r = p.repetition ? p.repetition[row] : p.repetition_all;
    s.p = p.presence ? p.presence[row] : p.presence_all;
    s.f = p.frequency ? p.frequency[row] : p.frequency_all;
    __syncthreads();
    // The tokens with a mark are listed, so that the work on them is spread over all threads: every kAdjThreads-th 16 bytes of counts are a thread's.
    constexpr int kLooks = ((SHORT ? kAdjLargest : kAdjLargestLong) + N) / PER / kAdjThreads + 1;
    uint32_t found[(kLooks + 3) / 4];          // eight bits a look
#pragma unroll
    for (int l = 0; l < (kLooks + 3) / 4; ++l) found[l] = 0u;
    int k = 0;
#pragma unroll
    for (int look = 0; look < kLooks; ++look) {
        const int i = tid + look * kAdjThreads;
        if (i >= words16) break;
        const uint4 n = reinterpret_cast<const uint4*>(count)[i];
        uint32_t bits;
        if (SHORT)
            bits = ((n.x & 0xFFFFu) ? 1u : 0u) | (n.x >> 16 ? 2u : 0u) | ((n.y & 0xFFFFu) ? 4u : 0u) | (n.y >> 16 ? 8u : 0u) | ((n.z & 0xFFFFu) ? 16u : 0u) | (n.z >> 16 ? 32u : 0u) |
                   ((n.w & 0xFFFFu) ? 64u : 0u) | (n.w >> 16 ? 128u : 0u);
        else
            bits = (n.x ? 1u : 0u) | (n.y ? 2u : 0u) | (n.z ? 4u : 0u) | (n.w ? 8u : 0u);
        found[look / 4] |= bits << (look % 4 * 8);
        k += __popc(bits);
    }
    int upto = k, base = 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xFFFFFFFFu, upto, o);
        if (lane >= o) upto += up;
    }
    if (lane == 31 && upto) base = atomicAdd(&sm_list, upto);
    base = __shfl_sync(0xFFFFFFFFu, base, 31) + upto - k;
#pragma unroll
    for (int l = 0; l < (kLooks + 3) / 4; ++l)
        for (uint32_t left = found[l]; left; left &= left - 1u) {
            const int bit = __ffs(left) - 1;
            list[base++] = (uint16_t)(PER * (tid + (4 * l + (bit >> 3)) * kAdjThreads) + (bit & 7));
        }
    __syncthreads();
    // Their results over what the copy left: where out is the logits themselves, a logit that the mask allows is still there.
    const int n_list = sm_list, n_bias = sm_biases;
    for (int i = tid; i < n_list; i += kAdjThreads) {
        const int own = list[i], t = own - N + v0;
        const float x = Pack<T>::get(in[t]);
        const bool allowed = !mask || ((mask[t >> 5] >> (t & 31)) & 1);
        const uint32_t n = marked(own);
        float y = penalized<M>(x, n, s);
        if (n & M::kBiased) {
            float sum = 0.f;
            for (int j = 0; j < n_bias; ++j)
                if (ids[j] == own) sum += bias[j];
            y += sum;
        }
        out[t] = Pack<T>::put(allowed ? y : -INFINITY);
    }
}

template <typename T, int kAdjThreads>
int launch_adjust(const AdjustLogitsArgs& a, cudaStream_t stream) {
    constexpr int kLargest = kAdjThreads == 512 ? kAdjLargest : kAdjLargestLong;
    AdjParams p = {a.logits, a.ld, a.out, a.ldo, (const long long*)a.tokens, a.ldk, a.lengths, a.prompt_lengths, a.repetition, a.presence, a.frequency, (const long long*)a.bias_ids, a.bias,
                   a.ldb, a.mask, a.ldm, a.repetition_all, a.presence_all, a.frequency_all, a.V, a.max_tokens, a.n_bias, 0};
    // Segments of a row: as few as shared memory allows, since every one reads all of the row's tokens, unless SMs would have nothing to do; then as many as the last round of CTAs has room for
    // (64 rows of 151936 with 4096 tokens and 100 biases: 4 of 38912 in one round 15.8 us; with counts of 32 bits 9 of 17408 in two rounds 18.5, 10 of 16384 in three 20.5).
    // Counted as two CTAs of 512 threads an SM; histories near 8192 tokens beside thousands of biases take the shared memory of one, and a second round.
    const long long slots = 1024ll / kAdjThreads * sms_of_current_device();
    long long n = ((long long)a.V + kLargest - 1) / kLargest;
    const long long rounds = (a.rows * n + slots - 1) / slots, most = ((long long)a.V + 2047) / 2048;
    n = rounds * slots / a.rows > n ? rounds * slots / a.rows : n;
    if (n > most) n = most;
    p.seg = (int)(((a.V + n - 1) / n + 1023) / 1024 * 1024);
    static bool once[64] = {};
    int dev = 0;
    PLZ_CUDA_CHECK(cudaGetDevice(&dev));
    if (!once[dev & 63]) {
        PLZ_CUDA_CHECK(cudaFuncSetAttribute((adjust_logits_kernel<T, kAdjThreads>), cudaFuncAttributeMaxDynamicSharedMemorySize, (kLargest + 16) * (kAdjThreads == 512 ? 4 : 6) + kAdjBiases * 8));
        once[dev & 63] = true;
    }
    const long long listed = (a.lengths ? (long long)a.max_tokens : 0) + a.n_bias, room = listed < p.seg + Pack<T>::N ? listed : p.seg + Pack<T>::N;
    const size_t smem = (a.lengths && a.max_tokens > 0) || a.n_bias > 0 ? (size_t)(p.seg + 8) * (kAdjThreads == 512 ? 2 : 4) + (size_t)a.n_bias * 8 + (size_t)room * 2 : 0;
    PLZ_LAUNCH_CHAIN_BEHIND((adjust_logits_kernel<T, kAdjThreads>), dim3((a.V + p.seg - 1) / p.seg, a.rows), dim3(kAdjThreads), smem, stream, p);
    return PLZ_OK;
}

}  // namespace

int launch_adjust_logits(int dtype, const AdjustLogitsArgs& a, cudaStream_t stream) {
    // Long histories, which every CTA of a row reads, are read by fewer CTAs of twice the threads (8 rows of 151936 with 30000 tokens 13.3 -> 11.0 us; 64 rows with 4096 tokens 15.8, 20.9 that way).
    if (a.lengths && a.max_tokens > kAdjShort) return dtype == 1 ? launch_adjust<float, 1024>(a, stream) : launch_adjust<__nv_bfloat16, 1024>(a, stream);
    return dtype == 1 ? launch_adjust<float, 512>(a, stream) : launch_adjust<__nv_bfloat16, 512>(a, stream);
}

}  // namespace plz
