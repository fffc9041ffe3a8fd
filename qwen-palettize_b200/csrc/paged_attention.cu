// Attention of one new token per request over a paged key / value cache, requests of any lengths in one launch:  o = softmax(q K^T * scale) V.
//
// Bound by memory: a cached token and key / value head is 4 * head_dim bytes that are read once, for the 4 * G * head_dim operations of the G query heads that share them.
//
//   paged_attn_kernel  One CTA per SM. The work is a line of steps of 16 tokens (32 of 64-wide heads): requests in order, in each its key / value heads (and blocks of 16 query heads), in each
//     its tokens. Every warp takes an equal stretch of the line, whatever the lengths are: it finds its first request by a sum over the lengths that its CTA makes. The pages of a step's
//     tokens are asked for four steps ahead, its keys and values two steps ahead, all by cp.async through a ring of the warp's own, which goes on over the ends of heads and requests: nothing waits
//     between short requests, and there is no barrier until a CTA's warps meet at the end.
//     Scores and sums are mma.sync m16n8k16 on fragments read by ldmatrix: the query heads are the 16 rows, the tokens the columns. tcgen05 has 64 rows at least, for the 4 query heads of
//     a group here, and would need the warps to meet in every step; the tensor pipe is 28 % busy at the speed of memory as it is.
//     Weights are three bf16 terms of the fp32 value, all 24 bits of it (two terms, 16 bits, differed from the sums in fp32 in the last bit of 0.2 % of the results). With up to 8 query heads
//     the second terms are rows 8 to 15 of the same product and cost nothing, the third are a product of their own: 256 short requests 39.9 -> 41.0 us, long ones within 1 %.
//     The accumulators of the products cut what falls below their last bit instead of rounding it: after n steps about n 2^-24 of a sum is gone (32 requests of 131072 tokens, 3500 steps a warp:
//     2.1 % of the results off in their last bit). So a warp's sums of 32 steps are added to earlier ones in fp32, rounded to nearest, which a lane keeps for itself in the workspace: then as many
//     results are off as with sums in fp32 throughout (64 requests of up to 4096 tokens 0.06 %, 2 x 131072 0.07 %). Replayed, without / 64 / 32 / 16 / 8 steps: 99 / 99.6 / 101.3 / 103.8 / 105 us
//     and 166 / 169 / 172 / 176 / 178; a step's sums added by themselves 100 and 167, but 182 where 32 steps take 176 and none 169, with the clocks of sustained load. With heads of 256, those of a step.
//     The reference of the exponentials moves when a row's maximum has grown by more than 2^8.
//     A head that a warp finishes alone goes to `out`; parts meet in shared memory at the end, parts that cross CTAs go to the workspace, two per CTA at most.
//   paged_join_kernel  one block per CTA of the first kernel and query head of a group joins the parts of the head that began there and went on; most have nothing to do.
//
// Measured, replayed (query / key heads 32 / 8 of 128, pages of 16 or 64): 2 x 131072 tokens 169 to 172 us for 1.07 GB, 6.3 TB/s; 64 requests of up to 4096 tokens 101 us for 0.58 GB, 5.7 TB/s; 256 requests
// of up to 300 tokens, 16 / 16 heads of 64, 39 us for 0.16 GB; one request of 2049 tokens 8.6 us, a chain of latencies: lengths, pages, keys, two meetings, a second launch. Heads 8 / 2 of 256,
// 32 requests of up to 4096 tokens, 38 us for 0.12 GB; 32 / 2 of 128, 64 such requests, 44 us for 0.14 GB.
//   What is in flight matters (before the third term and the kept sums): three steps a warp (196 KB of copies per SM) 187 and 110 us for the first two, since SMs then starve one another (their times
//   spread over 73 to 95 us at equal work, which taking the work as it comes did not mend: its many parts cost as much as it gave); two steps (128 KB) 160 and 96; six warps of two steps 166 and 100.
#include "plz_launch.h"

namespace plz {
namespace {

constexpr int kSwitch = 2;               // steps that the change to another head counts on the line (0: 256 short requests 45 us; 1, 2: 37; 4: 39)
constexpr int kCut = 32;                 // steps after which a warp's sums are kept elsewhere and begun anew
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
    float4* kept; float* parts; int4* heads;      // workspace: sums that a warp keeps; parts, two of every CTA and one of each of its warps; {request, item in it, last CTA} of the head that goes on from every CTA
    int B, width, page, n_pages, Hq, Hkv, G, blocks, items;   // blocks of 16 query heads per key / value head, items = Hkv * blocks
    int shift;                           // log2(page), or -1
    float scale_log2e;
};

__device__ __forceinline__ float ex2f(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory"); }
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

constexpr int kMostTokens = 0x7FFFFFC0;     // of a request: steps are counted by rounding up, and a step's last token is computed before it is compared, both within 31 of the length

// tokens of a request that are attended to
__device__ __forceinline__ int tokens_of(const PagedParams& p, int len) {
    const long long room = min((long long)p.width * p.page, (long long)kMostTokens);
    return len < 0 ? 0 : (long long)len > room ? (int)room : len;
}

// a place on the line of steps, and how much of a warp's stretch is left from there on
template <int TOK>
struct Place {
    int b, item, t, n, len;     // request, item in it, step in the item, steps of the request's items, its tokens
    int left, ahead;            // ahead: the next request's length, asked for when this one was opened
    __device__ __forceinline__ void open(const PagedParams& p, int length) {
        len = tokens_of(p, length);
        n = (len + TOK - 1) / TOK;
        ahead = b + 1 < p.B ? p.lengths[b + 1] : 0;
    }
    __device__ __forceinline__ void next_item(const PagedParams& p) {
        t = 0;
        if (++item < p.items) return;
        item = 0;
        do {
            if (++b >= p.B) { left = 0; return; }
            open(p, ahead);
        } while (n == 0);
    }
    __device__ __forceinline__ void next(const PagedParams& p) {
        --left;
        if (++t < n) return;
        left -= kSwitch;
        if (left > 0) next_item(p);
    }
};

template <int D_, int GP_, int TOK_, int NW_, int NST_>
struct Cfg {
    static constexpr int D = D_, GP = GP_, TOK = TOK_, NW = NW_, NST = NST_;
    static constexpr int kTile = TOK * D * 2;                       // bytes of a step's keys, or values
    static constexpr int kStage = 2 * kTile;
    static constexpr int kFree = 227 * 1024 - NW * NST * kStage - (NW * 32 * 8 + NW * (2 * 16 + 2 * NST * 16 + NST * TOK * 4 + NST * 4 + 8)) - 256;    // shared memory without the rings and the rest
    static constexpr int kPitch = D + 4;                            // floats between rows of a part: D sums, maximum, sum of weights
    static constexpr int kPart = GP * kPitch;                       // floats
    static constexpr int kRing = NST * kStage;
    // the part that a warp ends with takes the place of its ring; the one that it began with lies behind the ring, as far as it has rows that fit
    static constexpr int kRows = kFree / NW / (kPitch * 4) < GP ? kFree / NW / (kPitch * 4) : GP;
    static constexpr int kWarp = kRing + kRows * kPitch * 4;        // a warp's shared memory
    static constexpr int kSmem = NW * kWarp;
    static_assert(kPart * 4 <= kRing, "the last part lies in the ring");
};
struct PartMeta { int b, item, flags, rest; };      // flags 1: valid, 2: holds the head's first step, 4: holds its last; rest: steps behind it

template <typename C>
__global__ void __launch_bounds__(C::NW * 32, 1)
paged_attn_kernel(const PagedParams p) {
    constexpr int D = C::D, GP = C::GP, TOK = C::TOK, NW = C::NW, NST = C::NST, NR = GP / 8, KS = D / 16, NT = TOK / 8, CH = D / 8, ROWS = 32 / CH;
    constexpr bool EACH = D == 256;          // a step's sums are added to the others as they come: keeping them elsewhere takes registers that there are not (32 requests of up to 4096 tokens 43 us, 38 this way)
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ long long sm_first[NW * 32], sm_sum[NW];      // sums ahead of every thread's requests in its warp, of the warps
    __shared__ PartMeta sm_meta[NW][2];
    __shared__ int4 sm_step[NW][2 * NST];           // {request, item, step, tokens} of the steps that are seen
    __shared__ int sm_page[NW][NST][TOK];           // and the pages of their tokens
    __shared__ uint32_t sm_mask[NW][NST];           // which tokens of a step that was asked for count
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, cta = blockIdx.x, ctas = gridDim.x;
    pdl_launch_dependents();
    pdl_wait();

    // ---- the line, and where this warp begins on it: a request is items * (steps + kSwitch) long, one without tokens 0
    auto size_of = [&](int len) { const int n = (len + TOK - 1) / TOK; return n ? n + kSwitch : 0; };
    const int W = ctas * NW;
    long long total, stretch;
    auto cut = [&](long long sum) {                 // every warp's stretch; CTA c works from the places c * NW * stretch on
        total = sum * p.items;
        stretch = max(total <= 0x7FFFFFFF - W ? (long long)(((int)total + W - 1) / W) : (total + W - 1) / W, 1ll);
    };
    Place<TOK> eye;
    bool empty = false;
    long long off;
    if (lane < 2) sm_meta[warp][lane].flags = 0;
    if (p.B <= 32) {
        // a lane a request, every warp for itself: one request of 2049 tokens, replayed, 0.6 us less than by the sums below
        const int len = lane < p.B ? tokens_of(p, p.lengths[lane]) : 0, size = size_of(len);
        long long upto = size;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xFFFFFFFFu, upto, o);
            if (lane >= o) upto += u;
        }
        empty = __any_sync(0xFFFFFFFFu, lane < p.B && size == 0);
        cut(__shfl_sync(0xFFFFFFFFu, upto, 31));
        const long long begin = (cta * NW + warp) * stretch;
        eye.left = (int)min(total - begin, stretch);
        // the last request that begins there or ahead; of several, all but it are empty
        const int who = __popc(__ballot_sync(0xFFFFFFFFu, (upto - size) * p.items <= begin)) - 1;
        off = begin - __shfl_sync(0xFFFFFFFFu, upto - size, who) * p.items;
        eye.b = who;
        eye.len = __shfl_sync(0xFFFFFFFFu, len, who);
        eye.n = (eye.len + TOK - 1) / TOK;
        eye.ahead = __shfl_sync(0xFFFFFFFFu, len, (who + 1) & 31);
    } else {
        const int per = (p.B + NW * 32 - 1) / (NW * 32), r0 = min(p.B, tid * per), r1 = min(p.B, r0 + per);
        long long mine = 0;
        for (int b = r0; b < r1; ++b) {
            const int size = size_of(tokens_of(p, p.lengths[b]));
            mine += size;
            empty |= size == 0;
        }
        long long upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xFFFFFFFFu, upto, o);
            if (lane >= o) upto += u;
        }
        sm_first[tid] = upto - mine;
        if (lane == 31) sm_sum[warp] = upto;
        empty = __syncthreads_or(empty);
        // lane w: the sum of the warps ahead of w; lane NW: all
        long long ahead = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) ahead += w < lane ? sm_sum[w] : 0;
        cut(__shfl_sync(0xFFFFFFFFu, ahead, NW));
        const long long begin = (cta * NW + warp) * stretch;
        eye.left = (int)min(total - begin, stretch);
        if (eye.left > 0) {
            // the thread whose requests hold that place, then the request
            const int group = __popc(__ballot_sync(0xFFFFFFFFu, lane < NW && ahead * p.items <= begin)) - 1;
            const long long base = __shfl_sync(0xFFFFFFFFu, ahead, group);
            const int who = group * 32 + __popc(__ballot_sync(0xFFFFFFFFu, (base + sm_first[group * 32 + lane]) * p.items <= begin)) - 1;
            off = begin - (base + sm_first[who]) * p.items;
            eye.b = who * per;
            while (true) {
                eye.open(p, p.lengths[eye.b]);
                const long long size = (long long)size_of(eye.len) * p.items;
                if (off < size) break;
                off -= size;
                ++eye.b;
            }
        }
    }
    if (eye.left > 0) {
        const int one = eye.n + kSwitch;
        eye.item = off <= 0x7FFFFFFF ? (int)off / one : (int)(off / one);
        eye.t = (int)(off - (long long)eye.item * one);
        if (eye.t >= eye.n) {
            eye.left -= one - eye.t;
            if (eye.left > 0) eye.next_item(p);
        }
    }

    auto first_part = [&](int w) { return p.G <= C::kRows ? reinterpret_cast<float*>(smem + w * C::kWarp + C::kRing) : p.parts + ((size_t)cta * (2 + NW) + 2 + w) * C::kPart; };
    uint8_t* const mine_smem = smem + warp * C::kWarp;
    const uint32_t ring = smem_u32(mine_smem);
    if (eye.left > 0) {
        int seen = 0;                    // steps whose pages are asked for; all of the stretch's in the end
        const int lt = lane & (TOK - 1);
        auto see = [&]() {
            if (eye.left <= 0) return;
            if (lane == 0) sm_step[warp][seen % (2 * NST)] = make_int4(eye.b, eye.item, eye.t, eye.len);
            const int tok = eye.t * TOK + lt;
            if (lane < TOK && tok < eye.len)
                copy4(smem_u32(&sm_page[warp][seen % NST][lt]), p.table + (long long)eye.b * p.ldt + (p.shift >= 0 ? tok >> p.shift : tok / p.page));
            ++seen;
            eye.next(p);
        };
        auto ask = [&](int step) {
            if (step >= seen) return;
            const int slot = step % NST;
            const int4 st = sm_step[warp][step % (2 * NST)];
            const int tok = st.z * TOK + lt, pg = sm_page[warp][slot][lt];
            const bool in_len = tok < st.w, ok = in_len && (unsigned)pg < (unsigned)p.n_pages;
            if (in_len && !ok && p.bad) *p.bad = 1;
            const uint32_t mask = __ballot_sync(0xFFFFFFFFu, ok);
            if (lane == 0) sm_mask[warp][slot] = mask;
            const int in = p.shift >= 0 ? tok & (p.page - 1) : tok % p.page;
            const unsigned off = ok ? (unsigned)pg * p.page16 + (unsigned)in * p.tok16 : 0u;
            const int head = p.blocks == 1 ? st.y : st.y / p.blocks, c0 = lane % CH;
            const __nv_bfloat16 *kb = p.k + head * D + c0 * 8, *vb = p.v + head * D + c0 * 8;
            const uint32_t dst = ring + slot * C::kStage;
#pragma unroll
            for (int i = 0; i < TOK / ROWS; ++i) {
                const int row = i * ROWS + lane / CH;
                const unsigned o = __shfl_sync(0xFFFFFFFFu, off, row);
                const bool good = (mask >> row) & 1u;
                const uint32_t d = dst + row * (D * 2) + ((c0 ^ (row & 7)) << 4);
                copy16(d, kb + (size_t)o * 8, good);
                copy16(d + C::kTile, vb + (size_t)o * 8, good);
            }
        };
        // pages are asked for 2 NST steps ahead, keys and values NST: a group is one step's keys and values and a later one's pages
#pragma unroll 1
        for (int i = 0; i < NST; ++i) see();
        copy_commit();
        copy_wait<0>();
        __syncwarp();
#pragma unroll 1
        for (int i = 0; i < NST; ++i) { ask(i); see(); copy_commit(); }

        uint32_t qf[KS][2 * NR];
        float acc[D / 8][4], m[NR], l[NR], m_kept[NR];
        bool fresh = true, from_start = false, kept = false;
        const int g = lane >> 2, c2 = (lane & 3) * 2;
        float4* const sums = p.kept + (size_t)(cta * NW + warp) * (GP * D / 4) + lane;
        // with one row a lane the second terms' sums, rows 8 to 15, go to those of the first ones
        auto one_row = [&]() {
            if constexpr (NR == 1) {
#pragma unroll
                for (int n = 0; n < D / 8; ++n) { acc[n][0] += acc[n][2]; acc[n][1] += acc[n][3]; }
            }
        };
        // float4 i of a lane's sums: two columns of both rows, or of one row in two blocks of columns
        constexpr int NS = D * NR / 16;
        auto half = [&](int i, int h) -> float* { return NR == 1 ? acc[2 * i + h] : acc[i] + 2 * h; };
        auto add_kept = [&]() {
            if (!kept) return;
            float f[NR];
#pragma unroll
            for (int r = 0; r < NR; ++r) f[r] = m_kept[r] == m[r] ? 1.f : ex2f(m_kept[r] - m[r]);
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                const float4 o = sums[i * 32];
                float *const a = half(i, 0), *const b = half(i, 1);
                a[0] += f[0] * o.x; a[1] += f[0] * o.y;
                b[0] += f[NR - 1] * o.z; b[1] += f[NR - 1] * o.w;
            }
        };
#pragma unroll 1
        for (int step = 0, slot = 0;; ++step) {
            const int4 st = sm_step[warp][step % (2 * NST)];
            const int hk = p.blocks == 1 ? st.y : st.y / p.blocks, h0 = (st.y - hk * p.blocks) * 16, heads = min(p.G - h0, 16);
            if (fresh) {
                fresh = false;
                from_start = st.z == 0;
                const __nv_bfloat16* qr = p.q + (long long)st.x * p.ldq + (long long)(hk * p.G + h0) * D + c2;
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
                kept = false;
            }
            if (!EACH && __builtin_expect((step + 1) % kCut == 0, 0)) {
                one_row();
                add_kept();
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    const float *const a = half(i, 0), *const b = half(i, 1);
                    sums[i * 32] = make_float4(a[0], a[1], b[0], b[1]);
                }
#pragma unroll
                for (int n = 0; n < D / 8; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
#pragma unroll
                for (int r = 0; r < NR; ++r) m_kept[r] = m[r];
                kept = true;
            }
            copy_wait<NST - 1>();
            __syncwarp();
            const uint32_t kt = ring + slot * C::kStage, vt = kt + C::kTile;
            const uint32_t mask = sm_mask[warp][slot];
            float s[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
            {
                const int row = (lane & 7) + ((lane >> 4) << 3), upper = (lane >> 3) & 1;
                const uint32_t base = kt + row * (D * 2);
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int n = 0; n < NT; n += 2) {
                        uint32_t b[4];
                        ldm4(b, base + n * 8 * (D * 2) + (((2 * ks + upper) ^ (lane & 7)) << 4));
                        if constexpr (NR == 1) {
                            mma(s[n], qf[ks][0], 0u, qf[ks][1], 0u, b[0], b[1]);
                            mma(s[n + 1], qf[ks][0], 0u, qf[ks][1], 0u, b[2], b[3]);
                        } else {
                            mma(s[n], qf[ks][0], qf[ks][1], qf[ks][2], qf[ks][3], b[0], b[1]);
                            mma(s[n + 1], qf[ks][0], qf[ks][1], qf[ks][2], qf[ks][3], b[2], b[3]);
                        }
                    }
            }
            // scaled scores, maxima of the rows over the tokens that count
            float top[NR];
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                top[r] = -INFINITY;
#pragma unroll
                for (int n = 0; n < NT; ++n)
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
            uint32_t hi[NT][NR], mid[NT][NR], lo[NT][NR];
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                const float ref = m[r] == -INFINITY ? 0.f : m[r];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float w[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        w[e] = (mask >> (n * 8 + c2 + e)) & 1u ? ex2f(s[n][2 * r + e] - ref) : 0.f;
                        l[r] += w[e];
                    }
                    auto term = [&]() {            // 8 bits of each, which are taken off
                        const uint32_t t = pack_bf16x2(w[0], w[1]);
                        w[0] -= __uint_as_float(t << 16);
                        w[1] -= __uint_as_float(t & 0xFFFF0000u);
                        return t;
                    };
                    hi[n][r] = term();
                    mid[n][r] = term();
                    lo[n][r] = pack_bf16x2(w[0], w[1]);
                }
            }
            {
                const int row = (lane & 7) + (((lane >> 3) & 1) << 3), upper = lane >> 4;
                const uint32_t base = vt + row * (D * 2);
#pragma unroll
                for (int n = 0; n < NT; n += 2)
#pragma unroll
                    for (int j = 0; j < D / 16; j += 2) {
                        // four independent products between two that add to the same sums
                        float sum[4][4];
                        uint32_t b[2][4];
#pragma unroll
                        for (int i = 0; i < 2; ++i) ldm4t(b[i], base + n * 8 * (D * 2) + (((2 * (j + i) + upper) ^ (lane & 7)) << 4));
                        if (EACH) {
#pragma unroll
                            for (int i = 0; i < 4; ++i)
#pragma unroll
                                for (int e = 0; e < 4; ++e) sum[i][e] = 0.f;
                        }
                        auto add = [&](uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) mma(EACH ? sum[i] : acc[2 * j + i], a0, a1, a2, a3, b[i >> 1][2 * (i & 1)], b[i >> 1][2 * (i & 1) + 1]);
                        };
                        if constexpr (NR == 1) {
                            add(hi[n][0], mid[n][0], hi[n + 1][0], mid[n + 1][0]);
                            add(lo[n][0], 0u, lo[n + 1][0], 0u);
                        } else {
                            add(hi[n][0], hi[n][1], hi[n + 1][0], hi[n + 1][1]);
                            add(mid[n][0], mid[n][1], mid[n + 1][0], mid[n + 1][1]);
                            add(lo[n][0], lo[n][1], lo[n + 1][0], lo[n + 1][1]);
                        }
                        if (EACH) {
#pragma unroll
                            for (int i = 0; i < 4; ++i)
#pragma unroll
                                for (int e = 0; e < 4; ++e) acc[2 * j + i][e] += sum[i][e];
                        }
                    }
            }
            const bool over = step + 1 == seen, done = (st.z + 1) * TOK >= st.w;
            __syncwarp();
            ask(step + NST);
            see();
            copy_commit();
            slot = slot + 1 == NST ? 0 : slot + 1;
            if (done || over) {
                // rows r of this lane: query head g + 8 r
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], 1);
                    l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], 2);
                }
                one_row();
                add_kept();
                if (done && from_start) {
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        if (g + 8 * r >= heads) continue;
                        const float inv = 1.f / l[r];
                        __nv_bfloat16* o = p.out + (long long)st.x * p.ldo + (long long)(hk * p.G + h0 + g + 8 * r) * D + c2;
#pragma unroll
                        for (int n = 0; n < D / 8; ++n) *reinterpret_cast<uint32_t*>(o + n * 8) = pack_bf16x2(acc[n][2 * r] * inv, acc[n][2 * r + 1] * inv);
                    }
                } else {
                    // the part that a warp ends with goes to the place of its ring, into which nothing comes any more, the one that it began with, while the ring is at work, behind it
                    float* const part = over ? reinterpret_cast<float*>(mine_smem) : first_part(warp);
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        if (g + 8 * r >= heads) continue;
                        float* row = part + (g + 8 * r) * C::kPitch;
#pragma unroll
                        for (int n = 0; n < D / 8; ++n) *reinterpret_cast<float2*>(row + n * 8 + c2) = make_float2(acc[n][2 * r], acc[n][2 * r + 1]);
                        if (c2 == 0) *reinterpret_cast<float2*>(row + D) = make_float2(m[r], l[r]);
                    }
                    if (lane == 0) sm_meta[warp][over] = PartMeta{st.x, st.y, 1 | (from_start ? 2 : 0) | (done ? 4 : 0), (st.w + TOK - 1) / TOK - st.z - 1};
                }
                if (over) break;
                fresh = true;
            }
        }
        copy_wait<0>();
    }
    __syncthreads();

    // ---- the parts of this CTA, in order: those of one head follow one another. A warp takes a head and one of its rows at a time.
    auto part_at = [&](int i) -> const float* { return i & 1 ? reinterpret_cast<const float*>(smem + (i >> 1) * C::kWarp) : first_part(i >> 1); };
    const PartMeta own = lane < 2 * NW ? sm_meta[lane >> 1][lane & 1] : PartMeta{0, 0, 0, 0};
    const uint32_t valid = __ballot_sync(0xFFFFFFFFu, own.flags & 1), starts = __ballot_sync(0xFFFFFFFFu, (own.flags & 3) == 3) | (valid & -valid);
    const uint32_t ends = __ballot_sync(0xFFFFFFFFu, (own.flags & 5) == 5), begun = __ballot_sync(0xFFFFFFFFu, (own.flags & 3) == 3);
    if (tid == (NW - 1) * 32) p.heads[cta] = make_int4(0, 0, -1, 0);
    int turn = 0;
    for (uint32_t todo = starts; todo; todo &= todo - 1) {
        const int i = __ffs(todo) - 1, upper = todo & (todo - 1) ? __ffs(todo & (todo - 1)) - 1 : 32;
        const uint32_t run = valid & ~((1u << i) - 1u) & (upper == 32 ? 0xFFFFFFFFu : (1u << upper) - 1u);
        const int e = 31 - __clz(run);
        const bool first = (begun >> i) & 1u, last = (ends >> e) & 1u;
        const int b = __shfl_sync(0xFFFFFFFFu, own.b, i), item = __shfl_sync(0xFFFFFFFFu, own.item, i), rest = __shfl_sync(0xFFFFFFFFu, own.rest, e);
        const int hk = p.blocks == 1 ? item : item / p.blocks, h0 = (item - hk * p.blocks) * 16, heads = min(p.G - h0, 16);
        if (warp == NW - 1 && lane == 0 && first && !last) {
            // the head ends `rest` steps behind this CTA's stretches: the CTA that holds the last of them
            const long long at = (long long)(cta + 1) * NW * stretch + rest - 1, size = NW * stretch;
            p.heads[cta] = make_int4(b, item, at <= 0x7FFFFFFF ? (int)at / (int)size : (int)(at / size), 0);
        }
        float* const to = p.parts + ((size_t)cta * (2 + NW) + (first ? 1 : 0)) * C::kPart;
        for (int row = 0; row < heads; ++row, turn = turn + 1 == NW ? 0 : turn + 1) {
            if (turn != warp) continue;
            // lane j: part j's maximum and sum of weights
            float2 ml = make_float2(-INFINITY, 0.f);
            if ((run >> lane) & 1u) ml = *reinterpret_cast<const float2*>(part_at(lane) + row * C::kPitch + D);
            float top = ml.x;
#pragma unroll
            for (int o = 1; o < 2 * NW; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
            top = __shfl_sync(0xFFFFFFFFu, top, i);
            const float f = ml.x == top ? 1.f : ex2f(ml.x - top);
            float l = (run >> lane) & 1u ? f * ml.y : 0.f;
#pragma unroll
            for (int o = 1; o < 2 * NW; o <<= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, o);
            l = __shfl_sync(0xFFFFFFFFu, l, i);
#pragma unroll
            for (int n = 0; n < (D + 127) / 128; ++n) {
                const int d = n * 128 + lane * 4;
                float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
                const int at = row * C::kPitch + (d < D ? d : 0);
                for (uint32_t left = run; left;) {
                    // four at a time; past the last one that one again, without weight
                    int j[4];
                    float fj[4];
                    float4 v[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        j[k] = left ? __ffs(left) - 1 : j[k > 0 ? k - 1 : 0];
                        fj[k] = left ? 1.f : 0.f;
                        left &= left - 1u;
                        v[k] = *reinterpret_cast<const float4*>(part_at(j[k]) + at);
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        fj[k] *= __shfl_sync(0xFFFFFFFFu, f, j[k]);
                        o.x += fj[k] * v[k].x; o.y += fj[k] * v[k].y; o.z += fj[k] * v[k].z; o.w += fj[k] * v[k].w;
                    }
                }
                if (d >= D) continue;
                if (first && last) {
                    const float inv = 1.f / l;
                    *reinterpret_cast<uint2*>(p.out + (long long)b * p.ldo + (long long)(hk * p.G + h0 + row) * D + d) =
                        make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
                } else {
                    *reinterpret_cast<float4*>(to + row * C::kPitch + d) = o;
                }
            }
            if (!(first && last) && lane == 0) *reinterpret_cast<float2*>(to + row * C::kPitch + D) = make_float2(top, l);
        }
    }

    // ---- requests without tokens, and lengths that there cannot be
    for (int b = empty || p.bad ? cta : p.B; b < p.B; b += ctas) {
        const int len = p.lengths[b];
        if (tid == 0 && p.bad && len != tokens_of(p, len)) *p.bad = 1;
        if (!empty || tokens_of(p, len) > 0) continue;
        for (int x = tid * 8; x < p.Hq * D; x += NW * 256) *reinterpret_cast<uint4*>(p.out + (long long)b * p.ldo + x) = make_uint4(0u, 0u, 0u, 0u);
    }
}

// out = (sum_i 2^(m_i - m) o_i) / (sum_i 2^(m_i - m) l_i) over the parts i of a head, m the largest m_i: the second part of the CTA where the head began, the first ones of those
// behind it. One block per such CTA and query head of the item; its warps take the parts in turns, all loads of a warp's turn at once, and meet in shared memory.
// One sequence of 2049 tokens, 18 parts a head: 11 us with a thread per four sums of all heads.
constexpr int kJoinWarps = 8;
template <int D>
__global__ void __launch_bounds__(kJoinWarps * 32)
paged_join_kernel(const PagedParams p, int part, int per_cta) {
    constexpr int kPitch = D + 4, N = (D + 127) / 128, kTurn = 4;       // float4s of a lane; parts of a warp's turn
    __shared__ float4 sm_o[kJoinWarps][N][32];
    __shared__ float2 sm_ml[kJoinWarps];
    pdl_launch_dependents();
    pdl_wait();
    const int cta = blockIdx.x, row = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int4 h = p.heads[cta];
    if (h.z <= cta) return;
    const int hk = h.y / p.blocks, h0 = (h.y - hk * p.blocks) * 16, count = h.z - cta + 1;
    if (row >= min(p.G - h0, 16)) return;
    const size_t step = (size_t)per_cta * part;
    const float* const rest = p.parts + cta * step + row * kPitch;      // CTA cta + i: i steps on
    const float* const first = rest + part;
    float top = -INFINITY, l = 0.f;
    float4 o[N];
#pragma unroll
    for (int n = 0; n < N; ++n) o[n] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = warp; i0 < count; i0 += kJoinWarps * kTurn) {
        float2 ml[kTurn];
        float4 v[kTurn][N];
#pragma unroll
        for (int t = 0; t < kTurn; ++t) {
            const int i = i0 + t * kJoinWarps;
            if (i >= count) break;
            const float* part = i ? rest + i * step : first;
            ml[t] = *reinterpret_cast<const float2*>(part + D);
#pragma unroll
            for (int n = 0; n < N; ++n)
                if (n * 128 + lane * 4 < D) v[t][n] = *reinterpret_cast<const float4*>(part + n * 128 + lane * 4);
        }
#pragma unroll
        for (int t = 0; t < kTurn; ++t) {
            if (i0 + t * kJoinWarps >= count) break;
            const float to = fmaxf(top, ml[t].x), f = top == to ? 1.f : ex2f(top - to), g = ml[t].x == to ? 1.f : ex2f(ml[t].x - to);
            top = to;
            l = l * f + ml[t].y * g;
#pragma unroll
            for (int n = 0; n < N; ++n) {
                o[n].x = o[n].x * f + v[t][n].x * g; o[n].y = o[n].y * f + v[t][n].y * g;
                o[n].z = o[n].z * f + v[t][n].z * g; o[n].w = o[n].w * f + v[t][n].w * g;
            }
        }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) sm_o[warp][n][lane] = o[n];
    if (lane == 0) sm_ml[warp] = make_float2(top, l);
    __syncthreads();
    for (int x = threadIdx.x; x < D; x += kJoinWarps * 32) {
        float m = -INFINITY, sum = 0.f, w = 0.f;
#pragma unroll
        for (int i = 0; i < kJoinWarps; ++i) m = fmaxf(m, sm_ml[i].x);
#pragma unroll
        for (int i = 0; i < kJoinWarps; ++i) {
            if (i >= count) break;
            const float f = sm_ml[i].x == m ? 1.f : ex2f(sm_ml[i].x - m);
            sum += f * reinterpret_cast<const float*>(sm_o[i])[x];
            w += f * sm_ml[i].y;
        }
        p.out[(long long)h.x * p.ldo + (long long)(hk * p.G + h0 + row) * D + x] = __float2bfloat16_rn(sum / w);
    }
}

template <typename C>
int launch_paged(const PagedParams& p, int ctas, cudaStream_t stream) {
    static bool once[64] = {};
    int dev = 0;
    PLZ_CUDA_CHECK(cudaGetDevice(&dev));
    if (!once[dev & 63]) { PLZ_CUDA_CHECK(cudaFuncSetAttribute(paged_attn_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem)); once[dev & 63] = true; }
    PLZ_LAUNCH_CHAIN_BEHIND(paged_attn_kernel<C>, dim3(ctas), dim3(C::NW * 32), (size_t)C::kSmem, stream, p);
    PLZ_LAUNCH_CHAIN_BEHIND(paged_join_kernel<C::D>, dim3(ctas, p.G < 16 ? p.G : 16), dim3(kJoinWarps * 32), 0, stream, p, C::kPart, C::NW + 2);
    return PLZ_OK;
}

}  // namespace

// warps of a CTA, query heads of a part
static int warps_of(int d) { return d == 256 ? 4 : 8; }
static int rows_of(int Hq, int Hkv) { return Hq / Hkv > 8 ? 16 : 8; }
// floats of a CTA's parts, two of the CTA's and one of each warp's, and of the sums that its warps keep
static long long part_floats(int Hq, int Hkv, int d) { return (long long)(warps_of(d) + 2) * rows_of(Hq, Hkv) * (d + 4); }
static long long kept_floats(int Hq, int Hkv, int d) { return d == 256 ? 0 : (long long)warps_of(d) * rows_of(Hq, Hkv) * d; }

long long paged_attn_ws_bytes(int Hq, int Hkv, int head_dim) {
    return (long long)sms_of_current_device() * ((part_floats(Hq, Hkv, head_dim) + kept_floats(Hq, Hkv, head_dim)) * (long long)sizeof(float) + (long long)sizeof(int4));
}

int launch_paged_attn(const PagedAttnArgs& a, void* ws, long long ws_bytes, cudaStream_t stream) {
    if (ws_bytes < paged_attn_ws_bytes(a.Hq, a.Hkv, a.head_dim)) { set_last_error("attn_decode_paged: workspace of %lld bytes is too small", ws_bytes); return PLZ_ERR_WORKSPACE; }
    const int ctas = sms_of_current_device();
    PagedParams p = {};
    p.q = (const __nv_bfloat16*)a.q; p.ldq = a.ldq; p.k = (const __nv_bfloat16*)a.k_pages; p.v = (const __nv_bfloat16*)a.v_pages;
    p.page16 = (unsigned)(a.page_stride / 8); p.tok16 = (unsigned)(a.tok_stride / 8);
    p.table = a.table; p.ldt = a.ldt; p.lengths = a.lengths; p.out = (__nv_bfloat16*)a.out; p.ldo = a.ldo; p.bad = a.bad;
    p.kept = (float4*)ws;
    p.parts = (float*)ws + ctas * kept_floats(a.Hq, a.Hkv, a.head_dim);
    p.heads = (int4*)(p.parts + ctas * part_floats(a.Hq, a.Hkv, a.head_dim));
    p.B = a.B; p.width = a.width; p.page = a.page_size; p.n_pages = a.n_pages; p.Hq = a.Hq; p.Hkv = a.Hkv; p.G = a.Hq / a.Hkv;
    p.blocks = (p.G + 15) / 16; p.items = a.Hkv * p.blocks;
    p.shift = -1;
    if ((a.page_size & (a.page_size - 1)) == 0) { p.shift = 0; while ((1 << p.shift) < a.page_size) ++p.shift; }
    p.scale_log2e = a.scale * kLog2e;
    // more than eight query heads share a key: every term of the weights is a product of its own
    const bool wide = p.G > 8;
    if (a.head_dim == 64) return wide ? launch_paged<Cfg<64, 16, 32, 8, 2>>(p, ctas, stream) : launch_paged<Cfg<64, 8, 32, 8, 2>>(p, ctas, stream);
    if (a.head_dim == 128) return wide ? launch_paged<Cfg<128, 16, 16, 8, 2>>(p, ctas, stream) : launch_paged<Cfg<128, 8, 16, 8, 2>>(p, ctas, stream);
    return wide ? launch_paged<Cfg<256, 16, 16, 4, 2>>(p, ctas, stream) : launch_paged<Cfg<256, 8, 16, 4, 2>>(p, ctas, stream);
}

}  // namespace plz
