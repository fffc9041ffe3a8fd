// What a request's settings do to its logits before a token is picked: penalties for tokens that occurred, biases of single tokens, a grammar's mask.
//
//   x = x > 0 ? x / r : x * r  for tokens that occur;  x - f * c - p  for those that occur c > 0 times behind the prompt;  + biases;  -inf where the mask has a 0.
//
// Bound by memory (a logit read and written once) from a few rows on. One CTA takes a segment of a row: it counts the row's tokens that fall into the segment in shared memory (exact and in any
// order), and then streams the segment once, 16 bytes a thread and access. A token with a bias is marked in its count; who meets the mark walks the row's list of biases, so that
// several biases of one token are added in the order of the list whatever the threads do.
#include "plz_launch.h"

namespace plz {
namespace {

constexpr int kAdjThreads = 256;
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

__device__ __forceinline__ float adjusted(float x, uint32_t n, int t, const RowSettings& s, const AdjParams& p, int row) {
    if (n & (kSeen | kCount)) x = x > 0.f ? x / s.r : x * s.r;
    if (n & kCount) x = x - s.f * (float)(n & kCount) - s.p;
    if (n & kBiased) {
        const long long* ids = p.bias_ids + row * p.ldb;
        const float* b = p.bias + row * p.ldb;
        float sum = 0.f;
        for (int i = 0; i < p.n_bias; ++i)
            if (ids[i] == t) sum += b[i];
        x += sum;
    }
    return x;
}

// `seg` logits from the first 16-byte boundary of the row on; the few in front of it belong to the first segment
template <typename T>
__global__ void __launch_bounds__(kAdjThreads)
adjust_logits_kernel(const AdjParams p) {
    constexpr int N = Pack<T>::N;
    extern __shared__ uint32_t count[];
    const int row = blockIdx.y, tid = threadIdx.x;
    const T* in = (const T*)p.in + row * p.ld;
    T* out = (T*)p.out + row * p.ldo;
    const int head = (int)(((16u - (uint32_t)((uintptr_t)in & 15)) & 15u) / sizeof(T));
    const int s0 = blockIdx.x ? min(p.V, head + (int)blockIdx.x * p.seg) : 0, s1 = blockIdx.x + 1 == gridDim.x ? p.V : min(p.V, head + (int)(blockIdx.x + 1) * p.seg);
    pdl_launch_dependents();
    pdl_wait();
    RowSettings s;
    s.r = p.repetition ? p.repetition[row] : p.repetition_all;
    s.p = p.presence ? p.presence[row] : p.presence_all;
    s.f = p.frequency ? p.frequency[row] : p.frequency_all;
    const int n_tok = p.lengths ? min(max(p.lengths[row], 0), p.max_tokens) : 0, n_prompt = p.prompt_lengths ? max(p.prompt_lengths[row], 0) : 0;
    const bool marks = n_tok > 0 || p.n_bias > 0;
    if (marks) {
        for (int i = tid; i < s1 - s0; i += kAdjThreads) count[i] = 0;
        __syncthreads();
        const long long* tok = p.tokens + row * p.ldk;
        for (int i = tid; i < n_tok; i += kAdjThreads) {
            const long long t = tok[i] - s0;
            if (t < 0 || t >= s1 - s0) continue;
            if (i < n_prompt) atomicOr(count + t, kSeen); else atomicAdd(count + t, 1u);
        }
        const long long* ids = p.bias_ids + row * p.ldb;
        for (int i = tid; i < p.n_bias; i += kAdjThreads) {
            const long long t = ids[i] - s0;
            if (t >= 0 && t < s1 - s0) atomicOr(count + t, kBiased);
        }
        __syncthreads();
    }
    const int* mask = p.mask ? p.mask + row * p.ldm : nullptr;
    const int words = (p.V + 31) >> 5;
    const bool vec = (((uintptr_t)(out + head)) & 15) == 0;
    const int v0 = blockIdx.x ? s0 : min(head, s1), v1 = vec ? v0 + (s1 - v0) / N * N : v0;
    for (int i = v0 + tid * N; i < v1; i += kAdjThreads * N) {
        float x[N];
        Pack<T>::unpack(*reinterpret_cast<const uint4*>(in + i), x);
        if (marks) {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const uint32_t n = count[i - s0 + e];
                if (n) x[e] = adjusted(x[e], n, i + e, s, p, row);
            }
        }
        if (mask) {
            const int w = i >> 5;
            const uint32_t lo = mask[w], hi = w + 1 < words ? mask[w + 1] : 0u, bits = __funnelshift_r(lo, hi, i & 31);
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (!((bits >> e) & 1u)) x[e] = -INFINITY;
        }
        *reinterpret_cast<uint4*>(out + i) = Pack<T>::pack(x);
    }
    // what is not whole 16 bytes: in front of the first boundary, behind the last, or the segment where in and out lie differently
    const int front = v0 - s0, rest = front + s1 - v1;
    for (int j = tid; j < rest; j += kAdjThreads) {
        const int i = j < front ? s0 + j : v1 + j - front;
        float x = Pack<T>::get(in[i]);
        if (marks) {
            const uint32_t n = count[i - s0];
            if (n) x = adjusted(x, n, i, s, p, row);
        }
        if (mask && !((mask[i >> 5] >> (i & 31)) & 1)) x = -INFINITY;
        out[i] = Pack<T>::put(x);
    }
}

template <typename T>
int launch_adjust(const AdjustLogitsArgs& a, cudaStream_t stream) {
    AdjParams p = {a.logits, a.ld, a.out, a.ldo, (const long long*)a.tokens, a.ldk, a.lengths, a.prompt_lengths, a.repetition, a.presence, a.frequency, (const long long*)a.bias_ids, a.bias,
                   a.ldb, a.mask, a.ldm, a.repetition_all, a.presence_all, a.frequency_all, a.V, a.max_tokens, a.n_bias, 8192};
    const int segs = (a.V + p.seg - 1) / p.seg;
    PLZ_LAUNCH_CHAIN_BEHIND(adjust_logits_kernel<T>, dim3(segs, a.rows), dim3(kAdjThreads), (size_t)(p.seg + Pack<T>::N) * sizeof(uint32_t), stream, p);
    return PLZ_OK;
}

}  // namespace

int launch_adjust_logits(int dtype, const AdjustLogitsArgs& a, cudaStream_t stream) { return dtype == 1 ? launch_adjust<float>(a, stream) : launch_adjust<__nv_bfloat16>(a, stream); }

}  // namespace plz
