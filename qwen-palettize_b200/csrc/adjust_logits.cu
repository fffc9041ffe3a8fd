// What a request's settings do to its logits before a token is picked: penalties for tokens that occurred, biases of single tokens, a grammar's mask.
//
//   x = x > 0 ? x / r : x * r  for tokens that occur;  x - f * c - p  for those that occur c > 0 times behind the prompt;  + biases;  -inf where the mask has a 0.
//
// Bound by memory (a logit read and written once) from a few rows on. One CTA takes a segment of a row: it counts the row's tokens that fall into the segment in shared memory (exact and in any
// order), while the segment itself is on its way to registers, 16 bytes a thread and access. A warp lists the biases that fall into the segment in their order and marks their tokens' counts; who
// meets a mark walks that short list, so that several biases of one token are added in the order of the row's list whatever the threads do.
#include "plz_launch.h"

namespace plz {
namespace {

constexpr int kAdjThreads = 1024, kAdjUnits = 2;      // 16-byte units of a thread: all of a segment's logits are in registers at once
constexpr int kAdjBiases = 4096;         // of a row at most
constexpr uint32_t kSeen = 0x80000000u, kBiased = 0x40000000u, kCount = 0x3FFFFFFFu;

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
    __device__ __forceinline__ static void unpack(const uint4& v, float (&f)[4]) { f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w); }
    __device__ __forceinline__ static uint4 pack(const float (&f)[4]) { return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])); }
};
template <> struct Pack<__nv_bfloat16> {
    static constexpr int N = 8;
    __device__ __forceinline__ static float get(__nv_bfloat16 v) { return __bfloat162float(v); }
    __device__ __forceinline__ static __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
    __device__ __forceinline__ static void unpack(const uint4& v, float (&f)[8]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u); }
    }
    __device__ __forceinline__ static uint4 pack(const float (&f)[8]) { return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])); }
};

struct RowSettings { float r, p, f; };

// ids, bias: the segment's biases in the order of the row's list
__device__ __forceinline__ float adjusted(float x, uint32_t n, int t, const RowSettings& s, const int* ids, const float* bias, int n_bias) {
    if (n & (kSeen | kCount)) x = x > 0.f ? x / s.r : x * s.r;
    if (n & kCount) x = x - s.f * (float)(n & kCount) - s.p;
    if (n & kBiased) {
        float sum = 0.f;
        for (int i = 0; i < n_bias; ++i)
            if (ids[i] == t) sum += bias[i];
        x += sum;
    }
    return x;
}

// `seg` logits from the first 16-byte boundary of the row on; the few in front of it belong to the first segment
template <typename T>
__global__ void __launch_bounds__(kAdjThreads)
adjust_logits_kernel(const AdjParams p) {
    constexpr int N = Pack<T>::N;
    extern __shared__ __align__(16) uint32_t count[];
    __shared__ int sm_biases;
    int* const ids = reinterpret_cast<int*>(count + p.seg + 2 * N);
    float* const bias = reinterpret_cast<float*>(ids + p.n_bias);
    const int row = blockIdx.y, tid = threadIdx.x;
    const T* in = (const T*)p.in + row * p.ld;
    T* out = (T*)p.out + row * p.ldo;
    const int head = (int)(((16u - (uint32_t)((uintptr_t)in & 15)) & 15u) / sizeof(T));
    const int s0 = blockIdx.x ? min(p.V, head + (int)blockIdx.x * p.seg) : 0, s1 = blockIdx.x + 1 == gridDim.x ? p.V : min(p.V, head + (int)(blockIdx.x + 1) * p.seg);
    const bool vec = (((uintptr_t)(out + head)) & 15) == 0;
    const int v0 = blockIdx.x ? s0 : min(head, s1), v1 = vec ? v0 + (s1 - v0) / N * N : v0;      // whole 16-byte units, at most kAdjUnits a thread
    // segment t -> count[t - s0 + pad]: the first of a unit on a 16-byte boundary
    const int pad = (N - (v0 - s0) % N) % N;
    if (p.lengths || p.n_bias > 0)
        for (int i = tid; i < (pad + s1 - s0 + 3) / 4; i += kAdjThreads) reinterpret_cast<uint4*>(count)[i] = make_uint4(0u, 0u, 0u, 0u);
    pdl_launch_dependents();
    pdl_wait();
    // the segment's logits and masks are on their way while its tokens are counted
    const int* mask = p.mask ? p.mask + row * p.ldm : nullptr;
    const int words = (p.V + 31) >> 5;
    uint4 raw[kAdjUnits];
    uint32_t bits[kAdjUnits];
#pragma unroll
    for (int k = 0; k < kAdjUnits; ++k) {
        const int i = v0 + (k * kAdjThreads + tid) * N;
        bits[k] = 0xFFFFFFFFu;
        if (i >= v1) continue;
        raw[k] = *reinterpret_cast<const uint4*>(in + i);
        if (mask) {
            const int w = i >> 5;
            bits[k] = __funnelshift_r((uint32_t)mask[w], w + 1 < words ? (uint32_t)mask[w + 1] : 0u, i & 31);
        }
    }
    RowSettings s;
    s.r = p.repetition ? p.repetition[row] : p.repetition_all;
    s.p = p.presence ? p.presence[row] : p.presence_all;
    s.f = p.frequency ? p.frequency[row] : p.frequency_all;
    const int n_tok = p.lengths ? min(max(p.lengths[row], 0), p.max_tokens) : 0, n_prompt = p.prompt_lengths ? max(p.prompt_lengths[row], 0) : 0;
    const bool marks = n_tok > 0 || p.n_bias > 0;
    if (marks) {
        __syncthreads();
        const long long* tok = p.tokens + row * p.ldk;
        constexpr int U = 8;                   // tokens of a thread that are asked for together
        for (int i0 = tid; i0 < n_tok; i0 += kAdjThreads * U) {
            long long t[U];
#pragma unroll
            for (int u = 0; u < U; ++u) t[u] = i0 + u * kAdjThreads < n_tok ? tok[i0 + u * kAdjThreads] - s0 : -1;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (t[u] < 0 || t[u] >= s1 - s0) continue;
                if (i0 + u * kAdjThreads < n_prompt) atomicOr(count + pad + t[u], kSeen); else atomicAdd(count + pad + t[u], 1u);
            }
        }
        if (p.n_bias > 0 && tid >= kAdjThreads - 32) {
            // one warp keeps what falls into the segment, in its order
            const int lane = tid & 31;
            const long long* from = p.bias_ids + row * p.ldb;
            const float* value = p.bias + row * p.ldb;
            int n = 0;
            constexpr int U = 4;
            for (int i0 = lane; i0 - lane < p.n_bias; i0 += 32 * U) {
                long long t[U];
                float v[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const bool in = i0 + 32 * u < p.n_bias;
                    t[u] = in ? from[i0 + 32 * u] - s0 : -1;
                    v[u] = in ? value[i0 + 32 * u] : 0.f;
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const bool in = t[u] >= 0 && t[u] < s1 - s0;
                    const uint32_t all = __ballot_sync(0xFFFFFFFFu, in);
                    if (in) {
                        const int at = n + __popc(all & ((1u << lane) - 1u));
                        ids[at] = s0 + (int)t[u];
                        bias[at] = v[u];
                        atomicOr(count + pad + t[u], kBiased);
                    }
                    n += __popc(all);
                }
            }
            if (lane == 0) sm_biases = n;
        }
        __syncthreads();
    }
    const int n_bias = p.n_bias > 0 ? sm_biases : 0;
#pragma unroll
    for (int k = 0; k < kAdjUnits; ++k) {
        const int i = v0 + (k * kAdjThreads + tid) * N;
        if (i >= v1) continue;
        float x[N];
        Pack<T>::unpack(raw[k], x);
        if (marks) {
#pragma unroll
            for (int q = 0; q < N / 4; ++q) {
                const uint4 n4 = reinterpret_cast<const uint4*>(count)[(pad + i - s0) / 4 + q];
                const uint32_t n[4] = {n4.x, n4.y, n4.z, n4.w};
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (n[e]) x[4 * q + e] = adjusted(x[4 * q + e], n[e], i + 4 * q + e, s, ids, bias, n_bias);
            }
        }
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (!((bits[k] >> e) & 1u)) x[e] = -INFINITY;
        *reinterpret_cast<uint4*>(out + i) = Pack<T>::pack(x);
    }
    // what is not whole 16 bytes: in front of the first boundary, behind the last, or the segment where in and out lie differently
    const int front = v0 - s0, rest = front + s1 - v1;
    for (int j = tid; j < rest; j += kAdjThreads) {
        const int i = j < front ? s0 + j : v1 + j - front;
        float x = Pack<T>::get(in[i]);
        if (marks) {
            const uint32_t n = count[pad + i - s0];
            if (n) x = adjusted(x, n, i, s, ids, bias, n_bias);
        }
        if (mask && !((mask[i >> 5] >> (i & 31)) & 1)) x = -INFINITY;
        out[i] = Pack<T>::put(x);
    }
}

template <typename T>
int launch_adjust(const AdjustLogitsArgs& a, cudaStream_t stream) {
    AdjParams p = {a.logits, a.ld, a.out, a.ldo, (const long long*)a.tokens, a.ldk, a.lengths, a.prompt_lengths, a.repetition, a.presence, a.frequency, (const long long*)a.bias_ids, a.bias,
                   a.ldb, a.mask, a.ldm, a.repetition_all, a.presence_all, a.frequency_all, a.V, a.max_tokens, a.n_bias, 0};
    // the largest segment, whose tokens are read by the fewest CTAs, that still gives every SM one
    const int sms = sms_of_current_device();
    p.seg = kAdjThreads * kAdjUnits * Pack<T>::N;
    while (p.seg > 2048 && (long long)a.rows * ((a.V + p.seg - 1) / p.seg) < sms) p.seg /= 2;
    const size_t smem = (size_t)(p.seg + 2 * Pack<T>::N + 2 * a.n_bias) * sizeof(uint32_t);
    static bool once[64] = {};
    int dev = 0;
    PLZ_CUDA_CHECK(cudaGetDevice(&dev));
    if (!once[dev & 63]) {
        PLZ_CUDA_CHECK(cudaFuncSetAttribute(adjust_logits_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, ((kAdjThreads * kAdjUnits + 2) * Pack<T>::N + 2 * kAdjBiases) * (int)sizeof(uint32_t)));
        once[dev & 63] = true;
    }
    PLZ_LAUNCH_CHAIN_BEHIND(adjust_logits_kernel<T>, dim3((a.V + p.seg - 1) / p.seg, a.rows), dim3(kAdjThreads), smem, stream, p);
    return PLZ_OK;
}

}  // namespace

int launch_adjust_logits(int dtype, const AdjustLogitsArgs& a, cudaStream_t stream) { return dtype == 1 ? launch_adjust<float>(a, stream) : launch_adjust<__nv_bfloat16>(a, stream); }

}  // namespace plz
