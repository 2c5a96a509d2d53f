// Attention over the paged 8-bit KV cache: the new tokens' queries against all tokens of their request up to their own; here requests of few query
// rows (tq_paged_prompt.cu: many).
//
//   s = q . k scale,  o = sum softmax(s) v          q [tokens, heads * group, D] fp16, k and v code * 2^e of a page and head
//
// The query rows of a request and KV head are its new tokens times the heads of the group, token-major; there are 16 at most here, and
// paged_attn_kernel has room for 8 or 16 (8 NT; eight where no request has more): the decode step's kernel, bound by the bytes of the cache.  Every
// CTA streams an equal share of all (request, KV head, 64 tokens) units, whatever the requests' lengths, which only the device knows: it sums them up
// first and finds its share by itself.  An item (request, KV head) that ends in another CTA than it begins in is added up by paged_join_kernel, in
// order.
//
// One warp copies (bulk copies into a ring, an mbarrier per stage); four multiply, 16 tokens of a tile each, with a softmax of their own, so that
// they meet only at an item's end.  Products are mma.sync.m16n8k16 on halves with the tokens (then the dims) as the 16 rows and the query rows as the
// 8 columns, so that few query rows leave nothing idle; into the halves the codes go exactly: a byte b = code + 128 becomes the half 1024 + b by a
// byte permutation, and 1152 is taken off.  The order of the dims inside a product is free as long as both operands share it: a lane takes the 16
// dims of one 16-byte chunk.  (tcgen05 would need the operands in shared or tensor memory, behind a barrier for every tile, and 8 query rows leave
// most of its tile idle.)
//
// Rounding: products of halves are exact and summed in fp32; the softmax is fp32; the weights are rounded to halves for the second product (times
// 2^11, with a reference that lags by up to 2^4), their sum is taken before that.
//
// Measured, a new token each with 8 KV heads of 128 and a group of 5: 32 requests of 395 thousand tokens in all (809 MB) 148 us, 5.5 TB/s, 84 % of a
// copy's rate; two requests of 117 thousand in all 48 us, 76 %.  (Query rows as the 16 rows of the product, most of them empty: 226 and 78 us.)
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>

#include "tq_common.cuh"
#include "tq_paged.cuh"

namespace tq {

namespace {

using namespace paged_device;

constexpr int kTileTokens = 64;       // tokens of a unit
constexpr int kMulWarps = 4;
constexpr int kAttnThreads = 32 * (kMulWarps + 1);
// The reference maximum of a row moves only when a score exceeds it by 2^kSlack: a vote instead of a reduction for most tiles.  Weights are held
// times 2^kOffset and at most 2^15: halves that are normal numbers down to 2^-25 of the reference.
constexpr float kOffset = 11.f, kSlack = 4.f;

__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The 8 x 8 halves that a warp holds, two to a lane, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
// Two of the bytes of w (`which`: their places, with the 0x64 of a half behind each) as halves of code.
__device__ __forceinline__ uint32_t code_halves(uint32_t w, uint32_t which) {
    const uint32_t raw = __byte_perm(w, 0x64646464u, which);
    const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));   // 1152
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&raw), off);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// 2^-x, x byte r of `lower` (0 from 2^-127 on).
__device__ __forceinline__ float unit_ratio(uint32_t lower, int r) {
    return __int_as_float(max(127 - static_cast<int>(lower >> (8 * r) & 0xffu), 0) << 23);
}
// A request's part of the work, in units: its tiles (times the KV heads).
struct RequestWork {
    int row, start, count, held, lo, hi;   // tiles lo .. hi - 1 (none: not this kernel's)
    __device__ __forceinline__ void load(const PagedAttnArgs& a, int i) {
        row = a.b.rows[i];
        start = a.b.starts[i];
        count = a.b.starts[i + 1] - start;
        held = a.b.held[i];
        const int first = held - count;   // position of the first new token
        lo = a.window > 0 ? max(0, first - a.window + 1) / kTileTokens : 0;
        hi = count > 0 && count * a.group <= a.few_rows ? (held + kTileTokens - 1) / kTileTokens : lo;
    }
    // (A unit is some 8 KB of the cache at least, twice at most: all of them are a 32-bit number.)
    __device__ __forceinline__ unsigned int units(int heads) const { return static_cast<unsigned int>(heads) * static_cast<unsigned int>(hi - lo); }
};

// A CTA's share [u, end) of the units and where it stands in them: (request, KV head, tile), the tile running fastest.
struct Walker {
    RequestWork w;
    int i, head, tile;
    unsigned int left;   // units of the share that are still to do, this item's included
    __device__ __forceinline__ void place(const PagedAttnArgs& a, int request, unsigned int skip, unsigned int units) {
        i = request;
        left = units;
        w.load(a, i);
        while (skip >= w.units(a.heads)) {   // (the share begins inside a request that has units)
            skip -= w.units(a.heads);
            w.load(a, ++i);
        }
        const unsigned int tiles = static_cast<unsigned int>(w.hi - w.lo);
        tile = w.lo + static_cast<int>(skip % tiles);
        head = static_cast<int>(skip / tiles);
    }
    // Tiles of the present item that belong to the share.
    __device__ __forceinline__ int run() const { return static_cast<int>(min(static_cast<unsigned int>(w.hi - tile), left)); }
    // Behind that run; false at the share's end.
    __device__ __forceinline__ bool next(const PagedAttnArgs& a) {
        left -= static_cast<unsigned int>(run());
        if (left == 0) return false;
        if (++head == a.heads) {
            head = 0;
            do w.load(a, ++i);
            while (w.units(a.heads) == 0);
        }
        tile = w.lo;
        return true;
    }
};

// NT: query rows of an item in eights.
template <int D, int NT>
struct AttnShape {
    static constexpr int kRows = 8 * NT;
    static constexpr int kCtas = NT == 1 ? 3 : 2, kStages = NT == 1 ? 3 : 4;   // CTAs to an SM, tiles in a CTA's ring
    static constexpr int kTileBytes = kTileTokens * D;
    static constexpr int kScales = 4;   // pages in a tile at most
    static constexpr int kStageBytes = 2 * kTileBytes + 16 * kScales;
    static constexpr int kRowFloats = D + 4;
    static constexpr int kMergeBytes = kMulWarps * kRows * kRowFloats * 4;
    static constexpr int kSmem = kStages * kStageBytes + kMergeBytes;
    static constexpr int kPart = kRows * (D + 2);   // floats of a part: rows, then (maximum, sum) of each
};

// ONE: every request has one new token, so that its rows see the same and one unit of the values does for all of them.  Otherwise a window's or the
// drafts' end may lie between rows, and each has its own.  (Its own for single tokens too: 32 requests of 197 thousand tokens in all, 16 rows to
// each of 4 heads, 69.1 us for 67.1; of 395 thousand, 5 rows to each of 8, 135.2 for 133.9.)
template <int D, int NT, bool ONE>
__global__ void __launch_bounds__(kAttnThreads, AttnShape<D, NT>::kCtas) paged_attn_kernel(const __grid_constant__ PagedAttnArgs a) {
    using S = AttnShape<D, NT>;
    constexpr int kRows = S::kRows, kStages = S::kStages;
    extern __shared__ __align__(128) uint8_t s_mem[];
    __shared__ __align__(8) unsigned long long s_full[kStages], s_empty[kStages];
    __shared__ unsigned int s_sum[kAttnThreads + 1];
    __shared__ float s_ml[kMulWarps][kRows][2], s_vref[kMulWarps][kRows];
    __shared__ unsigned int s_abort;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) {
        for (int s = 0; s < kStages; ++s) {
            bar_init(smem_addr(&s_full[s]), 1);
            bar_init(smem_addr(&s_empty[s]), kMulWarps);
        }
        s_abort = 0;
        s_sum[0] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_wait_release();
    // units in front of each thread's requests (a plan that was refused has none, which is known only when they have been read)
    const int per = (a.sizes.n + kAttnThreads - 1) / kAttnThreads;
    {
        const int requests = planned(a.b.header, a.sizes, a.status).requests;
        unsigned int mine = 0;
        for (int i = tid * per; i < min(a.sizes.n, (tid + 1) * per); ++i) {
            RequestWork w;
            w.load(a, i);
            const unsigned int units = i < requests ? w.units(a.heads) : 0u;
            mine += units;
            if (units == 0u && blockIdx.x == 0)   // (its items, which no CTA begins)
                for (int k = i * a.heads; k < min((i + 1) * a.heads, a.join_items); ++k) a.joins[k].last = 0;
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned int t = __shfl_up_sync(0xffffffffu, mine, o);
            if (lane >= o) mine += t;
        }
        s_sum[tid + 1] = mine;
    }
    __syncthreads();
    unsigned int total = 0, before[kMulWarps + 1];
#pragma unroll
    for (int k = 0; k < kMulWarps + 1; ++k) {
        before[k] = total;
        total += s_sum[32 * (k + 1)];
    }
    const unsigned int ctas = min(gridDim.x, total), c = blockIdx.x;
    if (tid == 0 && a.join_items == 0) a.joins[c].last = 0;
    if (c >= ctas) return;
    const unsigned int share = total / ctas, extra = total - share * ctas;   // the first `extra` CTAs have one unit more
    const unsigned int u0 = c * share + min(c, extra), u1 = u0 + share + (c < extra ? 1u : 0u);
    Walker at;
    {
        // the thread's range of requests in which the share begins: the last whose sum in front is at most u0
        int lo = 0, hi = kAttnThreads;
        auto front = [&](int t) {
            unsigned int b = 0;
#pragma unroll
            for (int k = 0; k < kMulWarps + 1; ++k)
                if (k == t >> 5) b = before[k];
            return (t & 31) == 0 ? b : b + s_sum[t];
        };
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (front(mid) <= u0) lo = mid;
            else hi = mid;
        }
        at.place(a, lo * per, u0 - front(lo), u1 - u0);
    }

    if (warp == kMulWarps) {
        // ---- copies ----
        const int P = a.b.page_tokens, span = min(P, kTileTokens);   // tokens of a page in a tile
        const size_t block = paged_block_bytes(P, D);
        int known_row = -1, known_first = -1, known = 0;   // 32 entries of a row of the tables, one per lane
        uint32_t s = 0, phase = 0;
        bool ok = true, more = true;
        int issued = 0;
        while (ok && more) {
            const int tiles = at.run();
            for (int t = at.tile; ok && t < at.tile + tiles; ++t) {
                const int token = t * kTileTokens, here = min(kTileTokens, at.w.held - token), pages = (here + span - 1) / span;
                const int first = token / P;
                if (at.w.row != known_row || (first & ~31) != known_first) {
                    known_row = at.w.row;
                    known_first = first & ~31;
                    known = known_first + lane < a.b.max_pages ? a.b.tables[static_cast<size_t>(known_row) * a.b.max_pages + known_first + lane] : 0;
                }
                ok = bar_wait(smem_addr(&s_empty[s]), phase ^ 1, &s_abort);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                const uint32_t full = smem_addr(&s_full[s]);
                if (lane == 0) bar_expect(full, static_cast<uint32_t>(here * D * 2 + pages * 16));
                __syncwarp();
                // lanes 0 .. 3: keys of the pages, 4 .. 7: values, 8 .. 11: scales
                const int j = lane & 3, part = lane >> 2;
                const int page = __shfl_sync(0xffffffffu, known, (first + j) & 31);
                if (part < 3 && j < pages) {
                    const uint32_t bytes = static_cast<uint32_t>(min(span, here - j * span)) * D;
                    const uint8_t* const src = a.layer + (static_cast<size_t>(page) * a.heads + at.head) * block;
                    const uint32_t stage = smem_addr(s_mem) + s * S::kStageBytes;
                    const size_t in_page = static_cast<size_t>(P > kTileTokens ? token % P : 0) * D;
                    if (part == 0) bulk_copy(stage + j * span * D, src + in_page, bytes, full);
                    else if (part == 1) bulk_copy(stage + S::kTileBytes + j * span * D, src + static_cast<size_t>(P) * D + in_page, bytes, full);
                    else bulk_copy(stage + 2 * S::kTileBytes + 16 * j, src + 2 * static_cast<size_t>(P) * D, 16, full);
                }
                issued = min(issued + 1, kStages);
                if (++s == kStages) {
                    s = 0;
                    phase ^= 1;
                }
            }
            more = ok && at.next(a);
        }
        if (!ok) {
            if (lane == 0) {
                s_abort = 1;
                raise_status(a.status, kPagedWait);
            }
        }
        // Copies on their way land before the CTA's memory is another's: also where a multiplying warp gives up when all have been issued.  (The flag
        // does not cut this short.)
        unsigned int never = 0;
        for (int k = 0; k < issued; ++k) {
            if (s == 0) phase ^= 1;
            s = s == 0 ? kStages - 1 : s - 1;
            bar_wait(smem_addr(&s_full[s]), phase, &never);
        }
        return;
    }

    // ---- products ----
    const int g = lane >> 2, qd = lane & 3;
    const int P = a.b.page_tokens, span_shift = P >= kTileTokens ? 6 : P == 32 ? 5 : 4;
    const bool q_wide = ((reinterpret_cast<uintptr_t>(a.q) | static_cast<uintptr_t>(a.q_stride * 2)) & 7) == 0;
    const bool out_wide = ((reinterpret_cast<uintptr_t>(a.out) | static_cast<uintptr_t>(a.out_stride * 2)) & 15) == 0;
    uint32_t s = 0, phase = 0;
    bool more = true, alive = true;
    while (more) {
        const int rows = at.w.count * a.group;
        const int first_pos = at.w.held - at.w.count;
        // queries, the products' second operand: lane (g, qd) holds row g of each eight, of every 16-byte chunk c = qd + 4 j of codes the products 4
        // j .. 4 j + 3
        uint32_t qf[NT][D / 16][2];
        int pos[NT][2];   // of the scores' rows 2 qd, 2 qd + 1
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int row = min(8 * nt + g, rows - 1), token = row / a.group, hq = at.head * a.group + row - token * a.group;
            // (rows behind the last: the last again, nobody reads their results)
            const __half* const src = a.q + (at.w.start + token) * a.q_stride + static_cast<long>(hq) * D + 16 * qd;
#pragma unroll
            for (int j = 0; j < D / 64; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint2 v;
                    const __half* const p = src + 64 * j + 4 * k;
                    if (q_wide) v = *reinterpret_cast<const uint2*>(p);
                    else {
                        const __half2 x = __halves2half2(p[0], p[1]), y = __halves2half2(p[2], p[3]);
                        v = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
                    }
                    qf[nt][4 * j + k][0] = v.x;
                    qf[nt][4 * j + k][1] = v.y;
                }
#pragma unroll
            for (int e = 0; e < 2; ++e) pos[nt][e] = first_pos + min(8 * nt + 2 * qd + e, rows - 1) / a.group;
        }
        const int pos_min = first_pos, pos_max = first_pos + (rows - 1) / a.group;

        float o[NT][D / 16][4], m[NT][2], l[NT][2];
        // o is in units of the largest of the values' scales that its row has met: their exponents, a byte for each of the lane's rows (ONE: for all
        // of them, the lowest byte).
        uint32_t units = 0;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
            for (int u = 0; u < D / 16; ++u)
#pragma unroll
                for (int k = 0; k < 4; ++k) o[nt][u][k] = 0.f;
        }

        const int tiles = at.run();
        const bool begins = at.tile == at.w.lo, ends = at.tile + tiles == at.w.hi;
        for (int t = at.tile; t < at.tile + tiles; ++t) {
            alive = alive && __all_sync(0xffffffffu, bar_wait(smem_addr(&s_full[s]), phase, &s_abort));
            if (!alive) {   // (it still goes through the barriers with the others)
                if (lane == 0) {
                    s_abort = 1;
                    raise_status(a.status, kPagedWait);
                }
                break;
            }
            const uint8_t* const stage = s_mem + s * S::kStageBytes;
            const int w0 = t * kTileTokens + 16 * warp;   // this warp's first token
            if (w0 <= pos_max && (a.window <= 0 || w0 + 15 > pos_min - a.window)) {
                float2 scales = *reinterpret_cast<const float2*>(stage + 2 * S::kTileBytes + 16 * ((16 * warp) >> span_shift));
                if (!(scales.y < INFINITY)) scales = make_float2(__uint_as_float(0x7fc00000u), 0.f);   // values that are not numbers: the rows that see them
                // scores: tokens g (elements 0, 1) and g + 8 (2, 3), rows 2 qd and 2 qd + 1
                float sc[NT][4], odd[NT][4];   // (two chains of products)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int k = 0; k < 4; ++k) sc[nt][k] = odd[nt][k] = 0.f;
                const uint8_t* const keys = stage + 16 * warp * D;
#pragma unroll
                for (int j = 0; j < D / 64; ++j) {
                    const uint4 near = *reinterpret_cast<const uint4*>(keys + g * D + 16 * key_chunk<D>(g, qd + 4 * j));
                    const uint4 far = *reinterpret_cast<const uint4*>(keys + (g + 8) * D + 16 * key_chunk<D>(g, qd + 4 * j));
                    const uint32_t n4[4] = {near.x, near.y, near.z, near.w}, f4[4] = {far.x, far.y, far.z, far.w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t kf[4] = {code_halves(n4[k], 0x4140), code_halves(f4[k], 0x4140), code_halves(n4[k], 0x4342), code_halves(f4[k], 0x4342)};
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma_f16(k & 1 ? odd[nt] : sc[nt], kf, qf[nt][4 * j + k][0], qf[nt][4 * j + k][1]);
                    }
                }
                const float f = scales.x * a.scale_log2;
                const bool masks = w0 + 15 > pos_min || (a.window > 0 && w0 <= pos_max - a.window);
                // the values' exponent, for the rows that see some of these tokens: what a row does not see leaves its unit alone
                uint32_t value_units = __float_as_uint(scales.y) >> 23;
                if constexpr (!ONE) {
                    value_units *= 0x01010101u;
                    if (masks) {
#pragma unroll
                        for (int r = 0; r < 2 * NT; ++r)
                            if (w0 > pos[r >> 1][r & 1] || (a.window > 0 && w0 + 15 <= pos[r >> 1][r & 1] - a.window)) value_units &= ~(0xffu << (8 * r));
                    }
                }
                const uint32_t units_now = ONE ? max(units, value_units) : __vmaxu4(units, value_units);
                bool jump = units_now != units;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        float x = (sc[nt][k] + odd[nt][k]) * f;
                        if (masks) {
                            const int token = w0 + g + 8 * (k >> 1), p = pos[nt][k & 1];
                            if (token > p || (a.window > 0 && token <= p - a.window)) x = -INFINITY;
                        }
                        sc[nt][k] = x;
                        jump = jump || x > m[nt][k & 1] + kSlack;
                    }
                if (__any_sync(0xffffffffu, jump)) {
                    const uint32_t raised = units_now - units;   // (byte by byte)
                    units = units_now;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float top = fmaxf(sc[nt][e], sc[nt][2 + e]);
#pragma unroll
                            for (int b = 4; b < 32; b <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, b));
                            float down = 1.f;
                            if (top > m[nt][e] + kSlack) {
                                down = exp2_approx(m[nt][e] - top);   // (0 for the first)
                                m[nt][e] = top;
                            }
                            l[nt][e] *= down;
                            const float both = down * unit_ratio(raised, ONE ? 0 : 2 * nt + e);
#pragma unroll
                            for (int u = 0; u < D / 16; ++u) {
                                o[nt][u][e] *= both;
                                o[nt][u][2 + e] *= both;
                            }
                        }
                }
                const uint32_t lower = units - value_units;   // (byte by byte; of a row that sees nothing here the weights are 0)
                uint32_t pf[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float p[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float mk = m[nt][k & 1];
                        p[k] = exp2_approx(sc[nt][k] - ((mk == -INFINITY ? 0.f : mk) - kOffset));
                    }
                    l[nt][0] += p[0] + p[2];
                    l[nt][1] += p[1] + p[3];
                    // (row g, tokens 2 qd, 2 qd + 1 and 8 further on, as the second product wants them)
                    const float r0 = unit_ratio(lower, ONE ? 0 : 2 * nt), r1 = unit_ratio(lower, ONE ? 0 : 2 * nt + 1);
                    pf[nt][0] = transposed(pack_half2(p[0] * r0, p[1] * r1));
                    pf[nt][1] = transposed(pack_half2(p[2] * r0, p[3] * r1));
                }
                // values, transposed: lane (g, qd) takes the D / 8 dims of column g, of the tokens 2 qd, 2 qd + 1 and those 8 further on
                const uint8_t* const values = stage + S::kTileBytes + 16 * warp * D;
                constexpr int kWords = D / 32;   // 4 dims each
                uint32_t v[4][kWords];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int token = 2 * qd + (k & 1) + 8 * (k >> 1);
                    if constexpr (D == 128) {
                        const uint4 raw = *reinterpret_cast<const uint4*>(values + token * D + 16 * value_chunk<D>(token, g));
                        v[k][0] = raw.x; v[k][1] = raw.y; v[k][2] = raw.z; v[k][3] = raw.w;
                    } else {
                        const uint2 raw = *reinterpret_cast<const uint2*>(values + token * D + 16 * value_chunk<D>(token, g >> 1) + 8 * (g & 1));
                        v[k][0] = raw.x; v[k][1] = raw.y;
                    }
                }
#pragma unroll
                for (int w = 0; w < kWords; ++w)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        // bytes of two tokens side by side, of dims 2 h and 2 h + 1 of the word
                        const uint32_t near = __byte_perm(v[0][w], v[1][w], h ? 0x7362 : 0x5140), far = __byte_perm(v[2][w], v[3][w], h ? 0x7362 : 0x5140);
                        const uint32_t vf[4] = {code_halves(near, 0x4140), code_halves(near, 0x4342), code_halves(far, 0x4140), code_halves(far, 0x4342)};
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma_f16(o[nt][2 * w + h], vf, pf[nt][0], pf[nt][1]);
                    }
            }
            __syncwarp();
            if (lane == 0) bar_arrive(smem_addr(&s_empty[s]));
            if (++s == kStages) {
                s = 0;
                phase ^= 1;
            }
        }

        // ---- the four warps' sums together ----
        float* const s_o = reinterpret_cast<float*>(s_mem + kStages * S::kStageBytes);
        constexpr int kDims = D / 8;   // of a lane
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int b = 4; b < 32; b <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], b);
                const int r = 8 * nt + 2 * qd + e;
                float* const to = s_o + (warp * kRows + r) * S::kRowFloats + g * kDims;
#pragma unroll
                for (int u = 0; u < D / 16; u += 2)
                    *reinterpret_cast<float4*>(to + 2 * u) = make_float4(o[nt][u][e], o[nt][u][2 + e], o[nt][u + 1][e], o[nt][u + 1][2 + e]);
                if (g == 0) {
                    s_ml[warp][r][0] = m[nt][e];
                    s_ml[warp][r][1] = l[nt][e];
                    s_vref[warp][r] = __uint_as_float((units >> (ONE ? 0 : 8 * (2 * nt + e)) & 0xffu) << 23);
                }
            }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kMulWarps) : "memory");
        {
            constexpr int kEach = kRows * D / (32 * kMulWarps);   // dims of a thread
            const int r = tid / (D / kEach), d0 = tid % (D / kEach) * kEach;
            float top = -INFINITY, sum = 0.f, acc[kEach];
#pragma unroll
            for (int w = 0; w < kMulWarps; ++w) top = fmaxf(top, s_ml[w][r][0]);
#pragma unroll
            for (int d = 0; d < kEach; ++d) acc[d] = 0.f;
#pragma unroll
            for (int w = 0; w < kMulWarps; ++w) {
                // (a warp that saw nothing has zeros; one that met a NaN has no maximum, and its sum says so)
                const float mw = s_ml[w][r][0], x = mw == top || mw == -INFINITY ? 1.f : exp2_approx(mw - top), y = x * s_vref[w][r];
                sum = fmaf(s_ml[w][r][1], x, sum);
                const float* const from = s_o + (w * kRows + r) * S::kRowFloats + d0;
#pragma unroll
                for (int d = 0; d < kEach; d += 4) {
                    const float4 v = *reinterpret_cast<const float4*>(from + d);
                    acc[d] = fmaf(v.x, y, acc[d]);
                    acc[d + 1] = fmaf(v.y, y, acc[d + 1]);
                    acc[d + 2] = fmaf(v.z, y, acc[d + 2]);
                    acc[d + 3] = fmaf(v.w, y, acc[d + 3]);
                }
            }
            if (begins && ends) {
                if (r < rows) {
                    const int token = r / a.group, hq = at.head * a.group + r - token * a.group;
                    __half* const to = a.out + (at.w.start + token) * a.out_stride + static_cast<long>(hq) * D + d0;
                    const float inv = 1.f / sum;
#pragma unroll
                    for (int d = 0; d < kEach; d += 4) {
                        const uint2 four = make_uint2(pack_half2(acc[d] * inv, acc[d + 1] * inv), pack_half2(acc[d + 2] * inv, acc[d + 3] * inv));
                        if (out_wide) *reinterpret_cast<uint2*>(to + d) = four;
                        else {
                            to[d] = __ushort_as_half(static_cast<unsigned short>(four.x));
                            to[d + 1] = __ushort_as_half(static_cast<unsigned short>(four.x >> 16));
                            to[d + 2] = __ushort_as_half(static_cast<unsigned short>(four.y));
                            to[d + 3] = __ushort_as_half(static_cast<unsigned short>(four.y >> 16));
                        }
                    }
                    if (a.lse && d0 == 0)
                        a.lse[(at.w.start + token) * static_cast<long>(a.heads * a.group) + hq] = (top - kOffset + log2f(sum)) * 0.6931471805599453f;
                }
            } else {
                float* const part = a.partial + static_cast<long>(2 * c + (begins ? 1 : 0)) * S::kPart;
#pragma unroll
                for (int d = 0; d < kEach; d += 4) *reinterpret_cast<float4*>(part + r * D + d0 + d) = make_float4(acc[d], acc[d + 1], acc[d + 2], acc[d + 3]);
                if (d0 == 0) *reinterpret_cast<float2*>(part + kRows * D + 2 * r) = make_float2(top, sum);
            }
        }
        if (begins && tid == 0) {
            int last = 0;
            if (!ends) {
                // the CTA that holds the item's last unit
                const unsigned int unit = u1 - at.left + static_cast<unsigned int>(at.w.hi - at.tile) - 1, longer = extra * (share + 1);
                last = static_cast<int>(unit < longer ? unit / (share + 1) : extra + (unit - longer) / share);
            }
            if (a.join_items) {
                a.joins[at.i * a.heads + at.head] = {last, static_cast<int>(c), at.w.start, 0, rows, at.head};
            } else if (last) {
                a.joins[c] = {last, static_cast<int>(c), at.w.start, 0, rows, at.head};
            }
        }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kMulWarps) : "memory");
        more = at.next(a);
    }
}

// Parts of an item that several CTAs share, a CTA per item and row: eight warps take an eighth of the parts each, in the CTAs' order, and are added
// up in theirs.  It is bound by the latency of one load behind another, of which 8 parts' of a warp are on their way at once.  (A CTA per item: what
// one SM fetches from the L2 cache bounds it, 65 parts of a single request 13 -> 14.5 us.)
constexpr int kJoinWarps = 8;
template <int D, int NT>
__global__ void __launch_bounds__(32 * kJoinWarps) paged_join_kernel(const __grid_constant__ PagedAttnArgs a) {
    constexpr int kPart = AttnShape<D, NT>::kPart, kRows = 8 * NT, kEach = D / 32, kAtOnce = 8;
    __shared__ __align__(16) float s_acc[kJoinWarps][D];
    __shared__ float2 s_ml[kJoinWarps];
    pdl_wait_release();
    const PagedJoin join = a.joins[blockIdx.x];
    const int r = blockIdx.y, c = join.cta, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (join.last == 0 || r >= join.rows) return;
    const int parts = join.last - c + 1;
    const int k0 = parts * warp / kJoinWarps, k1 = parts * (warp + 1) / kJoinWarps;
    float acc[kEach] = {}, top = -INFINITY, sum = 0.f;
    for (int base = k0; base < k1; base += kAtOnce) {
        float2 ml[kAtOnce];
        float v[kAtOnce][kEach];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            const int part = min(base + k, k1 - 1);
            const float* const p = a.partial + static_cast<long>(2 * (c + part) + (part == 0 ? 1 : 0)) * kPart;
            ml[k] = *reinterpret_cast<const float2*>(p + kRows * D + 2 * r);
            if constexpr (kEach == 4) {
                const float4 f = *reinterpret_cast<const float4*>(p + r * D + 4 * lane);
                v[k][0] = f.x; v[k][1] = f.y; v[k][2] = f.z; v[k][3] = f.w;
            } else {
                const float2 f = *reinterpret_cast<const float2*>(p + r * D + 2 * lane);
                v[k][0] = f.x; v[k][1] = f.y;
            }
        }
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            if (base + k >= k1) continue;
            const float to = fmaxf(top, ml[k].x);
            const float y = top == to || top == -INFINITY ? 1.f : exp2_approx(top - to), x = ml[k].x == to || ml[k].x == -INFINITY ? 1.f : exp2_approx(ml[k].x - to);
            top = to;
            sum = fmaf(ml[k].y, x, sum * y);
#pragma unroll
            for (int d = 0; d < kEach; ++d) acc[d] = fmaf(v[k][d], x, acc[d] * y);
        }
    }
#pragma unroll
    for (int d = 0; d < kEach; ++d) s_acc[warp][kEach * lane + d] = acc[d];
    if (lane == 0) s_ml[warp] = make_float2(top, sum);
    __syncthreads();
    const int d = threadIdx.x;
    if (d >= D) return;
    top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) top = fmaxf(top, s_ml[w].x);
    float all = 0.f, value = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) {
        const float x = s_ml[w].x == top || s_ml[w].x == -INFINITY ? 1.f : exp2_approx(s_ml[w].x - top);
        all = fmaf(s_ml[w].y, x, all);
        value = fmaf(s_acc[w][d], x, value);
    }
    const int token = r / a.group, hq = join.head * a.group + r - token * a.group;
    a.out[(join.token + token) * a.out_stride + static_cast<long>(hq) * D + d] = __float2half_rn(value / all);
    if (a.lse && d == 0) a.lse[(join.token + token) * static_cast<long>(a.heads * a.group) + hq] = (top - kOffset + log2f(all)) * 0.6931471805599453f;
}

static_assert(kFewRows <= AttnShape<128, 2>::kRows, "a request's rows are one item");
template <int D, int NT>
void launch_typed(PagedAttnArgs a, int max_rows, void* scratch, int sms, cudaStream_t st) {
    using S = AttnShape<D, NT>;
    const int ctas = sms * S::kCtas;
    // Items that there can be: where they are fewer than the CTAs each has its own entry, and the kernel behind as many CTAs.
    const long items = static_cast<long>(a.sizes.n) * a.heads;
    a.join_items = items <= ctas ? static_cast<int>(items) : 0;
    a.joins = static_cast<PagedJoin*>(scratch);
    a.partial = reinterpret_cast<float*>(static_cast<char*>(scratch) + (ctas * sizeof(PagedJoin) + 255) / 256 * 256);
    static std::atomic<unsigned long long> set{0};
    static std::atomic<unsigned long long> set_one{0};
    const bool one = a.sizes.most == 1;
    if (one) allow_shared_memory(paged_attn_kernel<D, NT, true>, S::kSmem, set_one);
    else allow_shared_memory(paged_attn_kernel<D, NT, false>, S::kSmem, set);
    // (Both ask for all of the SM's memory as shared memory: an SM changes its division only when it is empty.)
    const auto attend = [&](auto kernel) { launch_pdl_carved(kernel, dim3(static_cast<unsigned int>(ctas)), dim3(kAttnThreads), S::kSmem, 100, st, a); };
    one ? attend(paged_attn_kernel<D, NT, true>) : attend(paged_attn_kernel<D, NT, false>);
    launch_pdl_carved(paged_join_kernel<D, NT>, dim3(static_cast<unsigned int>(a.join_items ? a.join_items : ctas), static_cast<unsigned int>(std::min(S::kRows, max_rows))),
                      dim3(32 * kJoinWarps), 0, 100, st, a);
}
template <int D, int NT>
size_t scratch_of(int sms) {
    using S = AttnShape<D, NT>;
    const size_t ctas = static_cast<size_t>(sms) * S::kCtas;
    return (ctas * sizeof(PagedJoin) + 255) / 256 * 256 + ctas * 2 * S::kPart * sizeof(float);
}

}  // namespace

size_t paged_attn_scratch_bytes(int dim, int sms) {
    return dim == 64 ? std::max(scratch_of<64, 1>(sms), scratch_of<64, 2>(sms)) : std::max(scratch_of<128, 1>(sms), scratch_of<128, 2>(sms));
}
void launch_paged_attention(PagedAttnArgs a, int dim, int max_rows, void* scratch, int sms, cudaStream_t st) {
    // Room for eight rows where no request has more: half the products and registers of sixteen.
    const bool eight = max_rows <= 8;
    if (dim == 64) eight ? launch_typed<64, 1>(a, max_rows, scratch, sms, st) : launch_typed<64, 2>(a, max_rows, scratch, sms, st);
    else eight ? launch_typed<128, 1>(a, max_rows, scratch, sms, st) : launch_typed<128, 2>(a, max_rows, scratch, sms, st);
}

}  // namespace tq
