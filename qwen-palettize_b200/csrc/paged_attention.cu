// Attention of one new token per request over a paged key / value cache, requests of any lengths in one launch:  o = softmax(q K^T * scale) V.
//
// Bound by memory: a cached token and key / value head is 4 * head_dim bytes that are read once, for the 4 * G * head_dim operations of the G query heads that share them.
//
//   paged_attn_kernel  One CTA per SM. The work is a line of steps of 16 tokens: requests in order, in each its key / value heads (and blocks of 16 query heads), in each its
//     tokens. Every warp takes an equal stretch of the line, whatever the lengths are: it finds its first request by a sum over the lengths that its CTA makes. A warp asks for its
//     steps NST ahead with 16-byte cp.async copies through a ring of its own, which goes on over the ends of heads and requests, so nothing waits between short requests and there is no
//     barrier until a CTA's warps meet at the end. Scores and sums are mma.sync m16n8k16 on fragments read by ldmatrix: the query heads are the 16 rows, the tokens the columns. (tcgen05 has
//     64 rows at least, for 4 query heads here, and would need the warps to meet in every step; with 4 heads the products use an eighth of what mma.sync offers at the speed of memory.)
//     Weights are two bf16 terms, high and low part, of the fp32 value: 16 bits of it enter the product, so the result is as exact as its own rounding to bf16. With up to 8 query heads
//     the low parts are rows 8 to 15 of the same product and cost nothing.
//     The reference of the exponentials moves when a row's maximum has grown by more than 2^8.
//     A head that a warp finishes alone goes to `out`; parts meet in shared memory at the end, parts that cross CTAs go to the workspace, two per CTA at most.
//   paged_join_kernel  one CTA per CTA of the first kernel joins the parts of the head that began there and went on; most have nothing to do.
#include "plz_launch.h"

namespace plz {
namespace {

constexpr int kTok = 16;                 // tokens of a step
constexpr float kGrow = 8.f;             // exponents (base 2) that a maximum may grow before the reference moves
constexpr float kLog2e = 1.4426950408889634f;

struct PagedParams {
    const __nv_bfloat16* q; long long ldq;
    const __nv_bfloat16 *k, *v;
    unsigned page16, tok16;              // strides of pages and token rows in 16-byte units
    const int* table; long long ldt;
    const int* lengths;
    __nv_bfloat16* out; long long ldo;
    int* bad;
    float* parts; int4* heads;           // workspace: two parts per CTA; {request, item in it, last CTA of the head that goes on} per CTA
    int B, width, page, n_pages, Hq, Hkv, G, blocks, items;   // blocks of 16 query heads per key / value head, items = Hkv * blocks
    int shift;                           // log2(page), or -1
    float scale_log2e;
};

__device__ __forceinline__ float ex2f(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldm4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// tokens of a request that are attended to
__device__ __forceinline__ int tokens_of(const PagedParams& p, int b) {
    const long long room = (long long)p.width * p.page;
    const int len = p.lengths[b];
    return len < 0 ? 0 : (long long)len > room ? (int)room : len;
}

// a place on the line of steps
struct Place {
    int b, item, t, n, len;     // request, item in it, step in the item, steps of the request's items, its tokens
    __device__ __forceinline__ void open(const PagedParams& p) { len = tokens_of(p, b); n = (len + kTok - 1) / kTok; }
    __device__ __forceinline__ void next(const PagedParams& p) {
        if (++t < n) return;
        t = 0;
        if (++item < p.items) return;
        item = 0;
        do { ++b; if (b < p.B) open(p); } while (b < p.B && n == 0);
    }
};

template <int D_, int GP_, int NW_, int NST_>
struct Cfg {
    static constexpr int D = D_, GP = GP_, NW = NW_, NST = NST_;
    static constexpr int kStage = 2 * kTok * D * 2;                 // bytes of a step: keys, then values
    static constexpr int kPitch = D + 4;                            // floats between rows of a part: D sums, maximum, sum of weights
    static constexpr int kPart = GP * kPitch * 4;
    static constexpr int kWarp = NST * kStage + kPart;              // a warp's shared memory: ring, its first part; its last part takes the ring's place
    static constexpr int kSmem = NW * kWarp;
    static_assert(kPart <= NST * kStage, "the last part lies in the ring");
};
struct PartMeta { int b, item, flags, rest; };                      // flags 1: valid, 2: holds the head's first step, 4: holds its last; rest: steps behind it
struct Start { int b; long long off; };

template <typename C>
__global__ void __launch_bounds__(C::NW * 32, 1)
paged_attn_kernel(const PagedParams p) {
    constexpr int D = C::D, GP = C::GP, NW = C::NW, NST = C::NST, NR = GP / 8, KS = D / 16, CH = D / 8, ROWS = 32 / CH > 0 ? 32 / CH : 1;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ long long sm_sum[NW];
    __shared__ Start sm_start[NW];
    __shared__ PartMeta sm_meta[NW][2];
    __shared__ uint32_t sm_mask[NW][NST];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, cta = blockIdx.x, ctas = gridDim.x;
    pdl_launch_dependents();
    pdl_wait();

    // ---- the line, and where this CTA's warps begin on it
    const int per = (p.B + NW * 32 - 1) / (NW * 32), r0 = min(p.B, tid * per), r1 = min(p.B, r0 + per);
    long long mine = 0;
    for (int b = r0; b < r1; ++b) mine += (tokens_of(p, b) + kTok - 1) / kTok;
    long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xFFFFFFFFu, upto, o);
        if (lane >= o) upto += u;
    }
    if (lane == 31) sm_sum[warp] = upto;
    if (lane < 2) sm_meta[warp][lane].flags = 0;
    __syncthreads();
    long long total = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        if (w < warp) upto += sm_sum[w];
        total += sm_sum[w];
    }
    total *= p.items;
    const int act = (int)min((long long)ctas, (total + NW - 1) / NW);     // CTAs at work: each has a step at least
    if (cta < act) {
        const long long W = (long long)act * NW, first = (upto - mine) * p.items, last = upto * p.items;
        if (mine > 0) {
            for (int w = 0; w < NW; ++w) {
                const long long s = total * (cta * NW + w) / W;
                if (s < first || s >= last) continue;
                long long at = first;
                int b = r0, n;
                for (;; ++b) {
                    n = (tokens_of(p, b) + kTok - 1) / kTok;
                    if (s < at + (long long)n * p.items) break;
                    at += (long long)n * p.items;
                }
                sm_start[w].b = b;
                sm_start[w].off = s - at;
            }
        }
    }
    __syncthreads();

    const uint32_t ring = smem_u32(smem) + warp * C::kWarp;
    float* const part0 = reinterpret_cast<float*>(smem + warp * C::kWarp + NST * C::kStage);
    float* const part1 = reinterpret_cast<float*>(smem + warp * C::kWarp);
    if (cta < act) {
        const long long W = (long long)act * NW, s0 = total * (cta * NW + warp) / W, s1 = total * (cta * NW + warp + 1) / W;
        long long todo = s1 - s0;
        if (todo > 0) {
            Place at;
            at.b = sm_start[warp].b;
            at.open(p);
            at.item = (int)(sm_start[warp].off / at.n);
            at.t = (int)(sm_start[warp].off - (long long)at.item * at.n);
            Place ahead = at;
            long long to_ask = todo;
            // the lane's token of the step that is asked for next: page and row in it
            int pg = -1, in = 0;
            auto look = [&]() {
                const int tok = ahead.t * kTok + (lane & 15);
                pg = -1;
                if (to_ask > 0 && tok < ahead.len) {
                    const int j = p.shift >= 0 ? tok >> p.shift : tok / p.page;
                    in = tok - j * p.page;
                    pg = p.table[(long long)ahead.b * p.ldt + j];
                }
            };
            auto ask = [&](int slot) {
                if (to_ask > 0) {
                    const bool in_len = ahead.t * kTok + (lane & 15) < ahead.len, ok = in_len && (unsigned)pg < (unsigned)p.n_pages;
                    if (in_len && !ok && p.bad) *p.bad = 1;
                    const uint32_t mask = __ballot_sync(0xFFFFFFFFu, ok) & 0xFFFFu;
                    if (lane == 0) sm_mask[warp][slot] = mask;
                    const unsigned off = ok ? (unsigned)pg * p.page16 + (unsigned)in * p.tok16 : 0u;
                    const int head = ahead.item / p.blocks, c0 = lane % CH;
                    const uint32_t dst = ring + slot * C::kStage;
#pragma unroll
                    for (int i = 0; i < kTok / ROWS; ++i) {
                        const int row = i * ROWS + lane / CH;
                        const unsigned o = __shfl_sync(0xFFFFFFFFu, off, row);
                        const bool good = (mask >> row) & 1u;
                        const size_t src = (size_t)o * 8 + head * D + c0 * 8;
                        const uint32_t d = dst + row * (D * 2) + ((c0 ^ (row & 7)) << 4);
                        copy16(d, p.k + src, good);
                        copy16(d + kTok * D * 2, p.v + src, good);
                    }
                    if (--to_ask > 0) ahead.next(p);
                    look();
                }
                copy_commit();
            };
            look();
#pragma unroll
            for (int i = 0; i < NST; ++i) ask(i);

            uint32_t qf[KS][2 * NR];
            float acc[D / 8][4], m[NR], l[NR];
            bool fresh = true, from_start = at.t == 0;
            int slot = 0, which = 0;
            const int g = lane >> 2, c2 = (lane & 3) * 2;
            while (true) {
                const int hk = at.item / p.blocks, h0 = (at.item - hk * p.blocks) * 16, heads = min(p.G - h0, 16);
                if (fresh) {
                    fresh = false;
                    const __nv_bfloat16* qr = p.q + (long long)at.b * p.ldq + (long long)(hk * p.G + h0) * D + c2;
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                        for (int r = 0; r < NR; ++r)
#pragma unroll
                            for (int h = 0; h < 2; ++h)
                                qf[ks][r + NR * h] = g + 8 * r < heads ? *reinterpret_cast<const uint32_t*>(qr + (long long)(g + 8 * r) * D + ks * 16 + h * 8) : 0u;
#pragma unroll
                    for (int n = 0; n < D / 8; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
#pragma unroll
                    for (int r = 0; r < NR; ++r) { m[r] = -INFINITY; l[r] = 0.f; }
                }
                copy_wait<NST - 1>();
                __syncwarp();
                const uint32_t kt = ring + slot * C::kStage, vt = kt + kTok * D * 2;
                const uint32_t mask = sm_mask[warp][slot];
                float s[2][4];
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
                {
                    const int row = (lane & 7) + ((lane >> 4) << 3), odd = (lane >> 3) & 1;
                    const uint32_t base = kt + row * (D * 2);
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) {
                        uint32_t b[4];
                        ldm4(b, base + (((2 * ks + odd) ^ (lane & 7)) << 4));
                        if constexpr (NR == 1) {
                            mma(s[0], qf[ks][0], 0u, qf[ks][1], 0u, b[0], b[1]);
                            mma(s[1], qf[ks][0], 0u, qf[ks][1], 0u, b[2], b[3]);
                        } else {
                            mma(s[0], qf[ks][0], qf[ks][1], qf[ks][2], qf[ks][3], b[0], b[1]);
                            mma(s[1], qf[ks][0], qf[ks][1], qf[ks][2], qf[ks][3], b[2], b[3]);
                        }
                    }
                }
                // scaled scores, maxima of the rows over the tokens that count
                float top[NR];
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    top[r] = -INFINITY;
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            s[n][2 * r + e] *= p.scale_log2e;
                            if ((mask >> (n * 8 + c2 + e)) & 1u) top[r] = fmaxf(top[r], s[n][2 * r + e]);
                        }
                    top[r] = fmaxf(top[r], __shfl_xor_sync(0xFFFFFFFFu, top[r], 1));
                    top[r] = fmaxf(top[r], __shfl_xor_sync(0xFFFFFFFFu, top[r], 2));
                }
                bool moves = false;
#pragma unroll
                for (int r = 0; r < NR; ++r) moves |= top[r] > m[r] + kGrow;       // m = -inf: any score moves it
                if (__any_sync(0xFFFFFFFFu, moves)) {
                    float f[NR];
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        const float to = fmaxf(m[r], top[r]);
                        f[r] = m[r] == to ? 1.f : ex2f(m[r] - to);
                        m[r] = to;
                        l[r] *= f[r];
                    }
#pragma unroll
                    for (int n = 0; n < D / 8; ++n) {
                        acc[n][0] *= f[0]; acc[n][1] *= f[0];
                        acc[n][2] *= f[NR - 1]; acc[n][3] *= f[NR - 1];
                    }
                }
                uint32_t hi[2][NR], lo[2][NR];
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    const float ref = m[r] == -INFINITY ? 0.f : m[r];
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        float w[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            w[e] = (mask >> (n * 8 + c2 + e)) & 1u ? ex2f(s[n][2 * r + e] - ref) : 0.f;
                            l[r] += w[e];
                        }
                        hi[n][r] = pack_bf16x2(w[0], w[1]);
                        lo[n][r] = pack_bf16x2(w[0] - __uint_as_float(hi[n][r] << 16), w[1] - __uint_as_float(hi[n][r] & 0xFFFF0000u));
                    }
                }
                {
                    const int row = (lane & 7) + (((lane >> 3) & 1) << 3), odd = lane >> 4;
                    const uint32_t base = vt + row * (D * 2);
#pragma unroll
                    for (int j = 0; j < D / 16; ++j) {
                        uint32_t b[4];
                        ldm4t(b, base + (((2 * j + odd) ^ (lane & 7)) << 4));
                        if constexpr (NR == 1) {
                            mma(acc[2 * j], hi[0][0], lo[0][0], hi[1][0], lo[1][0], b[0], b[1]);
                            mma(acc[2 * j + 1], hi[0][0], lo[0][0], hi[1][0], lo[1][0], b[2], b[3]);
                        } else {
                            mma(acc[2 * j], hi[0][0], hi[0][1], hi[1][0], hi[1][1], b[0], b[1]);
                            mma(acc[2 * j + 1], hi[0][0], hi[0][1], hi[1][0], hi[1][1], b[2], b[3]);
                            mma(acc[2 * j], lo[0][0], lo[0][1], lo[1][0], lo[1][1], b[0], b[1]);
                            mma(acc[2 * j + 1], lo[0][0], lo[0][1], lo[1][0], lo[1][1], b[2], b[3]);
                        }
                    }
                }
                __syncwarp();
                ask(slot);
                slot = slot + 1 == NST ? 0 : slot + 1;
                --todo;
                const bool done = at.t + 1 == at.n;
                if (done || todo == 0) {
                    // rows r of this lane: query head g + 8 r
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], 1);
                        l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], 2);
                    }
                    if constexpr (NR == 1) {
#pragma unroll
                        for (int n = 0; n < D / 8; ++n) { acc[n][0] += acc[n][2]; acc[n][1] += acc[n][3]; }
                    }
                    if (done && from_start) {
#pragma unroll
                        for (int r = 0; r < NR; ++r) {
                            if (g + 8 * r >= heads) continue;
                            const float inv = 1.f / l[r];
                            __nv_bfloat16* o = p.out + (long long)at.b * p.ldo + (long long)(hk * p.G + h0 + g + 8 * r) * D + c2;
#pragma unroll
                            for (int n = 0; n < D / 8; ++n) *reinterpret_cast<uint32_t*>(o + n * 8) = pack_bf16x2(acc[n][2 * r] * inv, acc[n][2 * r + 1] * inv);
                        }
                    } else {
                        // a last part comes when nothing is left to arrive in the ring
                        which = from_start ? 1 : 0;
                        if (which) { copy_wait<0>(); __syncwarp(); }
                        float* part = which ? part1 : part0;
#pragma unroll
                        for (int r = 0; r < NR; ++r) {
                            float* row = part + (g + 8 * r) * C::kPitch;
#pragma unroll
                            for (int n = 0; n < D / 8; ++n) *reinterpret_cast<float2*>(row + n * 8 + c2) = make_float2(acc[n][2 * r], acc[n][2 * r + 1]);
                            if (c2 == 0) { row[D] = m[r]; row[D + 1] = l[r]; }
                        }
                        if (lane == 0) sm_meta[warp][which] = PartMeta{at.b, at.item, 1 | (from_start ? 2 : 0) | (done ? 4 : 0), at.n - at.t - 1};
                    }
                    if (todo == 0) break;
                    fresh = from_start = true;
                }
                at.next(p);
            }
            copy_wait<0>();
        }
    }
    __syncthreads();

    // ---- the parts of this CTA, in order
    auto part_at = [&](int i) { return reinterpret_cast<const float*>(smem + (i >> 1) * C::kWarp + (i & 1 ? 0 : NST * C::kStage)); };
    int4 goes_on = make_int4(0, 0, -1, 0);
    for (int i = 0; i < 2 * NW;) {
        const PartMeta a = sm_meta[i >> 1][i & 1];
        if (!(a.flags & 1)) { ++i; continue; }
        int e = i, flags = a.flags;
        for (int j = i + 1; j < 2 * NW && !(flags & 4); ++j) {
            const int f = sm_meta[j >> 1][j & 1].flags;
            if (f & 1) { e = j; flags |= f; }
        }
        const int hk = a.item / p.blocks, h0 = (a.item - hk * p.blocks) * 16, heads = min(p.G - h0, 16);
        const bool whole = (flags & 6) == 6;
        float* to = p.parts + (size_t)(2 * cta + (flags & 2 ? 1 : 0)) * GP * C::kPitch;
        for (int x = tid * 4; x < heads * D; x += NW * 128) {
            const int row = x / D, d = x - row * D;
            float top = -INFINITY;
            for (int j = i; j <= e; ++j)
                if (sm_meta[j >> 1][j & 1].flags & 1) top = fmaxf(top, part_at(j)[row * C::kPitch + D]);
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
            float l = 0.f;
            for (int j = i; j <= e; ++j) {
                if (!(sm_meta[j >> 1][j & 1].flags & 1)) continue;
                const float* part = part_at(j) + row * C::kPitch;
                const float m = part[D], f = m == top ? 1.f : ex2f(m - top);
                const float4 v = *reinterpret_cast<const float4*>(part + d);
                o.x += f * v.x; o.y += f * v.y; o.z += f * v.z; o.w += f * v.w;
                l += f * part[D + 1];
            }
            if (whole) {
                const float inv = 1.f / l;
                *reinterpret_cast<uint2*>(p.out + (long long)a.b * p.ldo + (long long)(hk * p.G + h0 + row) * D + d) =
                    make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
            } else {
                *reinterpret_cast<float4*>(to + row * C::kPitch + d) = o;
                if (d == 0) { to[row * C::kPitch + D] = top; to[row * C::kPitch + D + 1] = l; }
            }
        }
        if ((flags & 6) == 2) {
            // the head ends `rest` steps behind this CTA's stretch: the CTA that holds the last of them
            const long long end = total * (cta + 1) / act + sm_meta[e >> 1][e & 1].rest;
            goes_on = make_int4(a.b, a.item, (int)((end * act - 1) / total), 0);
        }
        i = e + 1;
    }
    if (tid == 0) p.heads[cta] = goes_on;

    // ---- requests without tokens
    for (int b = cta; b < p.B; b += ctas) {
        const int len = p.lengths[b];
        if (tid == 0 && p.bad && (len < 0 || len > (long long)p.width * p.page)) *p.bad = 1;
        if (tokens_of(p, b) > 0) continue;
        for (int x = tid * 8; x < p.Hq * D; x += NW * 256) *reinterpret_cast<uint4*>(p.out + (long long)b * p.ldo + x) = make_uint4(0u, 0u, 0u, 0u);
    }
}

// out = (sum_i 2^(m_i - m) o_i) / (sum_i 2^(m_i - m) l_i) over the parts i of a head, m the largest m_i: the second part of this CTA, the first ones of those behind it
template <int D>
__global__ void __launch_bounds__(256)
paged_join_kernel(const PagedParams p, int gp) {
    constexpr int kPitch = D + 4;
    pdl_launch_dependents();
    pdl_wait();
    const int cta = blockIdx.x;
    const int4 h = p.heads[cta];
    if (h.z <= cta) return;
    const int hk = h.y / p.blocks, h0 = (h.y - hk * p.blocks) * 16, heads = min(p.G - h0, 16);
    const size_t step = (size_t)2 * gp * kPitch;
    for (int x = threadIdx.x * 4; x < heads * D; x += 1024) {
        const int row = x / D, d = x - row * D;
        const float* const first = p.parts + (size_t)(2 * cta + 1) * gp * kPitch + row * kPitch;
        const float* const rest = p.parts + (size_t)2 * cta * gp * kPitch + row * kPitch;      // CTA cta + i: i steps on
        float top = first[D];
        for (int i = 1; i <= h.z - cta; ++i) top = fmaxf(top, rest[i * step + D]);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        float l = 0.f;
#pragma unroll 4
        for (int i = 0; i <= h.z - cta; ++i) {
            const float* part = i ? rest + i * step : first;
            const float m = part[D], f = m == top ? 1.f : ex2f(m - top);
            const float4 v = *reinterpret_cast<const float4*>(part + d);
            o.x += f * v.x; o.y += f * v.y; o.z += f * v.z; o.w += f * v.w;
            l += f * part[D + 1];
        }
        const float inv = 1.f / l;
        *reinterpret_cast<uint2*>(p.out + (long long)h.x * p.ldo + (long long)(hk * p.G + h0 + row) * D + d) = make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
    }
}

template <typename C>
int launch_paged(const PagedParams& p, int ctas, cudaStream_t stream) {
    PLZ_CUDA_CHECK(cudaFuncSetAttribute(paged_attn_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    PLZ_LAUNCH_CHAIN_BEHIND(paged_attn_kernel<C>, dim3(ctas), dim3(C::NW * 32), (size_t)C::kSmem, stream, p);
    PLZ_LAUNCH_CHAIN_BEHIND(paged_join_kernel<C::D>, dim3(ctas), dim3(256), 0, stream, p, C::GP);
    return PLZ_OK;
}

}  // namespace

static long long part_floats(int Hq, int Hkv, int d) { return (long long)(Hq / Hkv > 8 ? 16 : 8) * (d + 4); }

long long paged_attn_ws_bytes(int Hq, int Hkv, int head_dim) {
    return (long long)sms_of_current_device() * (2 * part_floats(Hq, Hkv, head_dim) * (long long)sizeof(float) + (long long)sizeof(int4));
}

int launch_paged_attn(const PagedAttnArgs& a, void* ws, long long ws_bytes, cudaStream_t stream) {
    if (ws_bytes < paged_attn_ws_bytes(a.Hq, a.Hkv, a.head_dim)) { set_last_error("attn_decode_paged: workspace of %lld bytes is too small", ws_bytes); return PLZ_ERR_WORKSPACE; }
    const int ctas = sms_of_current_device();
    PagedParams p = {};
    p.q = (const __nv_bfloat16*)a.q; p.ldq = a.ldq; p.k = (const __nv_bfloat16*)a.k_pages; p.v = (const __nv_bfloat16*)a.v_pages;
    p.page16 = (unsigned)(a.page_stride / 8); p.tok16 = (unsigned)(a.tok_stride / 8);
    p.table = a.table; p.ldt = a.ldt; p.lengths = a.lengths; p.out = (__nv_bfloat16*)a.out; p.ldo = a.ldo; p.bad = a.bad;
    p.parts = (float*)ws;
    p.heads = (int4*)((char*)ws + ctas * 2 * part_floats(a.Hq, a.Hkv, a.head_dim) * (long long)sizeof(float));
    p.B = a.B; p.width = a.width; p.page = a.page_size; p.n_pages = a.n_pages; p.Hq = a.Hq; p.Hkv = a.Hkv; p.G = a.Hq / a.Hkv;
    p.blocks = (p.G + 15) / 16; p.items = a.Hkv * p.blocks;
    p.shift = -1;
    if ((a.page_size & (a.page_size - 1)) == 0) { p.shift = 0; while ((1 << p.shift) < a.page_size) ++p.shift; }
    p.scale_log2e = a.scale * kLog2e;
    const bool wide = p.G > 8;
    if (a.head_dim == 64) return wide ? launch_paged<Cfg<64, 16, 8, 5>>(p, ctas, stream) : launch_paged<Cfg<64, 8, 8, 6>>(p, ctas, stream);
    if (a.head_dim == 128) return wide ? launch_paged<Cfg<128, 16, 8, 2>>(p, ctas, stream) : launch_paged<Cfg<128, 8, 8, 3>>(p, ctas, stream);
    return wide ? launch_paged<Cfg<256, 16, 4, 2>>(p, ctas, stream) : launch_paged<Cfg<256, 8, 4, 3>>(p, ctas, stream);
}

}  // namespace plz
