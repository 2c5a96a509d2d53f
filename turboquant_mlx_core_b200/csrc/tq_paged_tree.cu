// Attention over the paged 8-bit KV cache for trees of drafts: each of a request's new tokens sees the tokens in front of the new ones, its
// ancestors and itself (paged_tree_kernel in tq_paged_plan.cu numbers the nodes).
//
// A request's query rows (new tokens times the heads of the group, token-major) are some tens to some hundreds: too many for the vectors of a decode
// step's kernel, too few for the 256 rows of a prompt's.  So the products are turned around: the 128 rows of a tensor core product are tokens
// of the cache, its N columns query rows, and a product takes as long as there are rows.
//
//   S^T [128 x N]  = K [128 x D] (shared memory) . Q^T [D x N] (shared memory)       fp16 products, fp32 sums, in tensor memory; two in turn
//   P^T            = 2^(S^T f + e - c + 7)  fp16, to shared memory
//   O^T [D x N]   += V^T [D x 128] . P^T [128 x N]                                   V as it lies: its dims in rows
//
// Keys and values go to shared memory as halves of the codes alone: with a token to a thread, the key's scale is that thread's factor f, the value's its
// summand e, and neither needs the codes to be multiplied.  c is a row's reference, the largest score times value scale that it has seen (in
// powers of two), or up to 2^8 below it: a row moves to a new one only when a weight would exceed 2^15.  The sum of weights is kept without the
// value's scale, each thread's for its own tokens, in fp32.
//
//   warps 0-3, 4-7   softmax: a thread has a token; the first four warps the first N / 2 rows, the others the rest
//   warps 8, 9       one lane issues the scores' products, the values'
//   warp 10          walks the CTA's share and tells the others, item by item, what is next
//   warp 11          queries, of the next item as soon as there is room
//   warps 12-19      keys: 16 tokens of a tile each, from memory through registers to shared memory
//   warps 20-27      values
//
// Tiles in which every row sees everything take the quick way; where a row sees only part of a tile (the drafts themselves, a window's end), at an item's
// beginning, where references move and where scales lie far apart the careful way is taken, by all four warps of a half: they agree on new
// references through shared memory.  As in the other kernels every CTA, one to an SM, takes an equal share of all units, and an item that
// ends in another CTA than it begins in is added up behind, in order.
//
// Every wait is bounded; a warp that gives up flags it, all warps fall through to the end, where the tensor memory is freed.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>

#include "tq_common.cuh"
#include "tq_paged.cuh"
#include "tq_paged_mma.cuh"

namespace tq {

namespace {

using namespace paged_device;

constexpr int kTokens = 128;         // of a unit (MMA M)
constexpr int kSWarp = 8, kScheduleWarp = 10, kQueryWarp = 11, kKeyWarp = 12, kValueWarp = 20, kWarps = 28, kThreads = 32 * kWarps;
// Registers a thread after the warpgroups have split what the CTA was launched with: 896 threads of 72.
constexpr int kLaunchRegs = 72, kSoftmaxRegs = 136, kControlRegs = 40, kCodeRegs = 48;
static_assert(256 * kSoftmaxRegs + 128 * kControlRegs + 512 * kCodeRegs <= kThreads * kLaunchRegs, "the shares are the launch's");
constexpr int kItemUnits = 2;        // what an item's beginning and end cost, in units
constexpr int kStages = 2;           // of keys and of values, as halves
constexpr int kSlots = 4;            // tiles whose scales are kept
constexpr int kGroups = kTokens / 16;   // of a tile's tokens that are in one page: a warp's
constexpr float kOffset = 7.f, kLimit = 15.f;   // weights are held times 2^7, and at most 2^15
constexpr float kSumOffset = 24.f;   // sums of weights times 2^24: their terms span 2^-97 .. 2^92 whatever the values' scales
constexpr float kNone = -3e38f;      // reference of a row that has seen nothing
constexpr float kLeastScale = -60.f; // values of smaller scales (below 2^-53) count as 0: half of the least half is 2^-25
constexpr float kSpread = 60.f;      // of the values' scales on the quick way
constexpr uint32_t kTmemAll = 512;

template <int D, int N>
struct Shape {
    static constexpr uint32_t kRowGroup = 16 * D;                        // 8 tokens or rows: D / 8 core matrices of 128 bytes
    static constexpr uint32_t kPGroup = 16 * N;                          // 8 tokens of P^T: N / 8 core matrices
    static constexpr int kQStages = N <= 64 ? 2 : 1;
    static constexpr uint32_t kQBytes = N / 8 * kRowGroup, kTileBytes = kTokens / 8 * kRowGroup, kPBytes = kTokens / 8 * kPGroup;
    // (D = 64: the product of 128 rows reads eight dims' core matrices beyond a tile's last, which are P's: rows that nobody reads)
    static constexpr uint32_t kQ = 0, kK = kQStages * kQBytes, kV = kK + kStages * kTileBytes, kP = kV + kStages * kTileBytes, kSmem = kP + 2 * kPBytes;
    static constexpr int kHalf = N / 2;                                  // rows of a softmax thread
    static constexpr int kPart = N * (D + 2);                            // floats: [N][D], then (reference, sum) of each row
};

struct Request {
    int row, start, count, held, rows, lo, hi, blocks;
    template <int N>
    __device__ __forceinline__ void load(const PagedAttnArgs& a, int i) {
        row = a.b.rows[i];
        start = a.b.starts[i];
        count = a.b.starts[i + 1] - start;
        held = a.b.held[i];
        if (count > 0 && !a.b.nodes[start].good) count = 0;
        rows = count * a.group;
        blocks = (rows + N - 1) / N;
        hi = (held + kTokens - 1) / kTokens;
        lo = a.window > 0 ? max(0, held - count - a.window + 1) / kTokens : 0;
    }
    __device__ __forceinline__ int first() const { return held - count; }
    __device__ __forceinline__ long long item() const { return hi - lo + kItemUnits; }
    __device__ __forceinline__ long long units(const PagedAttnArgs& a) const { return count > 0 ? item() * blocks * a.heads : 0; }
};

// A CTA's share of the units: (request, KV head, block of rows, tile), the tile running fastest.  All lanes hold the same.
template <int N>
struct Walker {
    Request r;
    int i, n, head, block, tile;
    int before;          // units of kItemUnits that come in front of the present tile
    long long left;
    // The first request from `from` on with more than `skip` units behind those in front of it; `skip` becomes what is left of it.
    __device__ __forceinline__ bool find(const PagedAttnArgs& a, int from, long long& skip, int lane) {
        for (int base = from; base < n; base += 32) {
            Request x;
            x.load<N>(a, min(base + lane, n - 1));
            const long long mine = base + lane < n ? x.units(a) : 0;
            long long upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long t = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += t;
            }
            const unsigned int beyond = __ballot_sync(0xffffffffu, upto > skip);
            if (beyond) {
                const int src = __ffs(static_cast<int>(beyond)) - 1;
                skip -= __shfl_sync(0xffffffffu, upto - mine, src);
                i = base + src;
                r.load<N>(a, i);
                return true;
            }
            skip -= __shfl_sync(0xffffffffu, upto, 31);
        }
        return false;
    }
    __device__ __forceinline__ void place(const PagedAttnArgs& a, int from, int requests, long long skip, long long units, int lane) {
        n = requests;
        left = units;
        if (!find(a, from, skip, lane)) {   // (not with a share of units that exist)
            left = 0;
            return;
        }
        const long long item = static_cast<long long>(skip / r.item());
        const int in = static_cast<int>(skip - item * r.item());
        head = static_cast<int>(item / r.blocks);
        block = static_cast<int>(item - static_cast<long long>(head) * r.blocks);
        before = max(0, kItemUnits - in);
        tile = r.lo + max(0, in - kItemUnits);
    }
    // Tiles of the present item that belong to the share.
    __device__ __forceinline__ int run() const { return static_cast<int>(min(static_cast<long long>(r.hi - tile), max(0ll, left - before))); }
    __device__ __forceinline__ bool next(const PagedAttnArgs& a, int lane) {
        left -= before + run();
        if (left <= 0) return false;
        if (++block == r.blocks) {
            block = 0;
            if (++head == a.heads) {
                head = 0;
                long long none = 0;
                if (!find(a, i + 1, none, lane)) return false;
            }
        }
        tile = r.lo;
        before = kItemUnits;
        return left > before;
    }
};
// The part of an item that a CTA does, as the scheduling warp tells the others.
struct __align__(16) Segment {
    int row, start, first, held;   // of the request: row of the tables, first token, position of its first new token, tokens
    int rows, row0, head;          // its query rows, the first of this item
    int tile, tiles;               // (0: the end)
    int begins, ends;              // whether it holds the item's first and last tile
    int last;                      // the CTA in which the item ends
};
constexpr int kSegments = 4;
constexpr int kSegmentReaders = 8 + 2 + 1 + 16;   // warps: softmax, products, queries, keys and values

struct Bars {
    unsigned long long q_full[2], q_empty[2], s_full[2], p_full[2], o_done[2], k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages],
        vote[2], seg_full[kSegments], seg_empty[kSegments], done[2];
};

// Two of the bytes of w (`which`: their places, with the 0x64 of a half behind each) as halves of code: 1024 + byte, less 1152.
__device__ __forceinline__ uint32_t code_halves(uint32_t w, uint32_t which) {
    const uint32_t raw = __byte_perm(w, 0x64646464u, which);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&raw), __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&h);
}
// The largest of a warp's numbers, of those that are numbers and above kNone.
__device__ __forceinline__ float warp_max(float x) {
    const uint32_t b = __float_as_uint(fmaxf(x, kNone));
    const uint32_t top = __reduce_max_sync(0xffffffffu, b & 0x80000000u ? ~b : b | 0x80000000u);
    return __uint_as_float(top & 0x80000000u ? top & 0x7fffffffu : ~top);
}
// Sums over the warp's lanes of W numbers each: lane l's is of number l % W.
template <int W>
__device__ __forceinline__ float lane_sums(float (&v)[W], int lane) {
    if constexpr (W == 16) {
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], 16);
    }
#pragma unroll
    for (int s = W / 2; s > 0; s >>= 1) {
        const bool upper = (lane & s) != 0;
#pragma unroll
        for (int k = 0; k < s; ++k) {
            const float mine = upper ? v[k + s] : v[k], other = upper ? v[k] : v[k + s];
            v[k] = mine + __shfl_xor_sync(0xffffffffu, other, s);
        }
    }
    return v[0];
}

template <int D, int N>
__global__ void __launch_bounds__(kThreads, 1) paged_tree_attn_kernel(const __grid_constant__ PagedAttnArgs a) {
    using S = Shape<D, N>;
    constexpr int kHalf = S::kHalf, kChunk = kHalf < 32 ? kHalf : 32, kChunks = kHalf / kChunk;
    extern __shared__ __align__(1024) uint8_t s_mem[];
    __shared__ __align__(8) Bars s_bar;
    __shared__ long long s_sum[kWarps];
    __shared__ __align__(16) float2 s_scale[kSlots][kGroups];   // keys', values'
    __shared__ __align__(16) float s_ref[2][2][kHalf];          // [version][half]: minus a row's reference, and kOffset
    __shared__ __align__(16) Segment s_seg[kSegments];
    __shared__ unsigned int s_flag[2][4];                       // [half][tile]: a reference has to move
    __shared__ uint32_t s_tmem;
    __shared__ unsigned int s_abort;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    auto bar = [&](unsigned long long& b) { return smem_addr(&b); };
    if (tid == 0) {
        for (int k = 0; k < 2; ++k) {
            bar_init(bar(s_bar.q_full[k]), 1);
            bar_init(bar(s_bar.q_empty[k]), 1);
            bar_init(bar(s_bar.s_full[k]), 1);
            bar_init(bar(s_bar.p_full[k]), 8);
            bar_init(bar(s_bar.o_done[k]), 1);
            bar_init(bar(s_bar.vote[k]), 4);
            bar_init(bar(s_bar.done[k]), 1);
        }
        for (int k = 0; k < kStages; ++k) {
            bar_init(bar(s_bar.k_full[k]), kGroups);
            bar_init(bar(s_bar.k_empty[k]), 1);
            bar_init(bar(s_bar.v_full[k]), kGroups);
            bar_init(bar(s_bar.v_empty[k]), 1);
        }
        for (int k = 0; k < kSegments; ++k) {
            bar_init(bar(s_bar.seg_full[k]), 1);
            bar_init(bar(s_bar.seg_empty[k]), kSegmentReaders);
        }
        for (int k = 0; k < 8; ++k) s_flag[k >> 2][k & 3] = 0;
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_wait_release();
    int n = planned(a.b.header, a.sizes, a.status).requests;
    if (n > 0 && a.b.header->state != kPagedTree) {   // (a plan of the same sizes that has no trees)
        if (blockIdx.x == 0 && tid == 0) raise_status(a.status, kPagedOtherPlan);
        n = 0;
    }
    const int per = (n + kWarps - 1) / kWarps;
    {
        long long mine = 0;
        for (int i = warp * per + lane; i < min(n, (warp + 1) * per); i += 32) {
            Request r;
            r.load<N>(a, i);
            mine += r.units(a);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
        if (lane == 0) s_sum[warp] = mine;
    }
    __syncthreads();
    long long total = 0;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) total += s_sum[k];
    const long long ctas = min(static_cast<long long>(gridDim.x), total), c = blockIdx.x;
    if (tid == 0) a.joins[c].last = 0;
    if (c >= ctas) return;
    if (warp == kSWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)), "r"(kTmemAll) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        fence_before();
    }
    __syncthreads();
    fence_after();
    const uint32_t tmem = s_tmem, base = smem_addr(s_mem);
    constexpr uint32_t kO = 2 * N;   // column of O^T, behind two of S^T
    volatile unsigned int* const flag = &s_abort;
    bool ok = true;
    auto wait = [&](unsigned long long& b, uint32_t phase) {
        if (ok && !__all_sync(0xffffffffu, bar_wait(smem_addr(&b), phase, flag))) {
            ok = false;
            s_abort = 1;
        }
        return ok;
    };
    // The segments in turn; false behind the last.  `done_with` gives the last one back.
    uint32_t seg_n = 0;
    auto next_segment = [&]() { return wait(s_bar.seg_full[seg_n % kSegments], (seg_n / kSegments) & 1) && s_seg[seg_n % kSegments].tiles > 0; };
    auto done_with = [&]() {
        __syncwarp();
        if (lane == 0) bar_arrive(bar(s_bar.seg_empty[seg_n % kSegments]));
        ++seg_n;
    };

    if (warp < kSWarp) {
        // ---- softmax: a thread per token ----
        take_registers<kSoftmaxRegs>();
        const int half = warp >> 2, quarter = warp & 3, token_in = 32 * quarter + lane;
        const uint32_t lanes = static_cast<uint32_t>(quarter) << 21;   // this warp's 32 lanes of tensor memory
        const uint32_t t_s0 = tmem + lanes + half * kHalf, t_o = tmem + lanes + kO + half * kHalf;
        // this thread's eight rows of halves in P^T, and room of its warp's there for a number of each row while nothing else is
        uint8_t* const p_at = s_mem + S::kP + (token_in >> 3) * S::kPGroup + half * kHalf * 16 + (token_in & 7) * 16;
        auto room = [&](uint32_t buffer, int q) { return reinterpret_cast<float*>(s_mem + S::kP + buffer * S::kPBytes + 4 * q * S::kPGroup + half * kHalf * 16); };
        uint32_t done = 0, votes = 0;   // tiles so far; meetings of the four warps
        int version = 0;
        auto meet = [&]() {   // what the four warps wrote before is everyone's behind it
            __syncwarp();
            if (lane == 0) bar_arrive(bar(s_bar.vote[half]));
            return wait(s_bar.vote[half], votes++ & 1);
        };
        unsigned long long sum2[kHalf / 2];   // of this thread's tokens' weights, for each row
        while (next_segment()) {
            const Segment at = s_seg[seg_n % kSegments];
            // what the lane's rows of the half are: number, and position, of their nodes
            constexpr int kOwn = (kHalf + 31) / 32;
            int own_pre[kOwn], own_pos[kOwn];
#pragma unroll
            for (int k = 0; k < kOwn; ++k) {
                const int row = min(at.row0 + half * kHalf + 32 * k + lane, at.rows - 1);
                const PagedNode node = a.b.nodes[at.start + row / a.group];
                own_pre[k] = node.pre;
                own_pos[k] = at.first + node.depth;
            }
#pragma unroll
            for (int k = 0; k < kHalf / 2; ++k) sum2[k] = 0ull;
            __syncwarp();
            for (int k = lane; k < kHalf; k += 32) s_ref[version][half][k] = kOffset - kNone;
            __syncwarp();
            bool bare = true;                       // a row of the half has seen nothing
            float largest = kLeastScale;            // exponent of the values' scales so far
            for (int j = 0; j < at.tiles; ++j) {
                const uint32_t n = done + j, buffer = n & 1;
                if (!wait(s_bar.s_full[buffer], (n >> 1) & 1)) break;
                if (n >= 2 && !wait(s_bar.o_done[buffer], ((n >> 1) - 1) & 1)) break;   // (P^T's place)
                fence_after();
                const uint32_t t_s = t_s0 + buffer * N;
                uint8_t* const p_to = p_at + buffer * S::kPBytes;
                const int token = (at.tile + j) * kTokens + token_in;
                const float2 scale = s_scale[n & (kSlots - 1)][token_in >> 4];
                float most = kLeastScale, least = 200.f;
#pragma unroll
                for (int k = 0; k < kGroups; ++k) {
                    const float v = s_scale[n & (kSlots - 1)][k].y;
                    const float e = v < INFINITY ? static_cast<float>(static_cast<int>(__float_as_uint(v) >> 23) - 127) : 0.f;
                    most = fmaxf(most, e);
                    least = fminf(least, e);
                }
                largest = fmaxf(largest, most);
                const bool fine = scale.y < INFINITY;   // (values that are not numbers: the scores are none)
                const float f = fine ? scale.x < INFINITY ? fmaxf(scale.x * a.scale_log2, 1.1754944e-38f) : __uint_as_float(0x7fc00000u) : __uint_as_float(0x7fc00000u);
                const float e_true = fine ? static_cast<float>(static_cast<int>(__float_as_uint(scale.y) >> 23) - 127) : 0.f, e = fmaxf(e_true, kLeastScale);
                const int tile_end = (at.tile + j + 1) * kTokens;
                const bool masked = tile_end > at.first || (a.window > 0 && (at.tile + j) * kTokens < at.held - a.window);
                bool careful = masked || bare || least < kLeastScale || least < largest - kSpread;
                int summed = 0;   // chunks of rows whose sums have this tile's weights
                if (!careful) {
                    const float g = __int_as_float((127 + static_cast<int>(kSumOffset - kOffset - e)) << 23);
                    const unsigned long long f2 = pack2(f, f), e2 = pack2(e, e), g2 = pack2(g, g);
                    const float wild = 83.f + fminf(e, 0.f);   // a weight that the sum might not hold
                    bool moves = false, over = false;
#pragma unroll
                    for (int q = 0; q < kChunks; ++q) {
                        if (over) break;
                        uint32_t x[kChunk];
                        tmem_ld(t_s + q * kChunk, x);
                        tmem_ld_wait(x);
                        float top = -INFINITY;
                        const float* const ref = s_ref[version][half] + q * kChunk;
#pragma unroll
                        for (int k = 0; k < kChunk; k += 4) {
                            const float4 r4 = *reinterpret_cast<const float4*>(ref + k);
                            const float2 y = unpack2(add2(fma2(pack2(__uint_as_float(x[k]), __uint_as_float(x[k + 1])), f2, e2), pack2(r4.x, r4.y)));
                            const float2 z = unpack2(add2(fma2(pack2(__uint_as_float(x[k + 2]), __uint_as_float(x[k + 3])), f2, e2), pack2(r4.z, r4.w)));
                            top = fmaxf(fmaxf(top, fmaxf(y.x, y.y)), fmaxf(z.x, z.y));
                            x[k] = __float_as_uint(y.x);
                            x[k + 1] = __float_as_uint(y.y);
                            x[k + 2] = __float_as_uint(z.x);
                            x[k + 3] = __float_as_uint(z.y);
                        }
                        moves = moves || top > kLimit;
                        over = __any_sync(0xffffffffu, top > wild);
                        if (over) break;
#pragma unroll
                        for (int k = 0; k < kChunk; k += 8) {
                            uint32_t h[4];
#pragma unroll
                            for (int m = 0; m < 4; ++m) {
                                const float px = exp2_approx(__uint_as_float(x[k + 2 * m])), py = exp2_approx(__uint_as_float(x[k + 2 * m + 1]));
                                unsigned long long& to = sum2[(q * kChunk + k) / 2 + m];
                                to = fma2(pack2(px, py), g2, to);
                                h[m] = pack_half2(px, py);
                            }
                            *reinterpret_cast<uint4*>(p_to + (q * kChunk + k) * 16) = make_uint4(h[0], h[1], h[2], h[3]);
                        }
                        summed = q + 1;
                    }
                    if (__any_sync(0xffffffffu, moves) && lane == 0) s_flag[half][n & 3] = 1;
                }
                // (the flags of two tiles on: everyone has read them when they were those of two tiles ago)
                if (quarter == 0 && lane == 0) s_flag[half][(n + 2) & 3] = 0;
                if (!careful) {
                    if (!meet()) break;
                    careful = *const_cast<volatile unsigned int*>(&s_flag[half][n & 3]) != 0;
                }
                if (careful) {
                    // a token's place in its tree: rows whose nodes' numbers are lo .. lo + span see it, from a position on that the window leaves
                    int lo = 0, place = token;
                    unsigned int span = 0xffffffffu;
                    bool there = token < at.held;
                    if (there && token >= at.first) {
                        const PagedNode node = a.b.nodes[at.start + token - at.first];
                        lo = node.pre;
                        span = static_cast<unsigned int>(node.last - node.pre);
                        place = at.first + node.depth;
                    }
                    auto sees = [&](int row) {   // (of the half; by all lanes)
                        const int pre = __shfl_sync(0xffffffffu, own_pre[row >> 5 < kOwn ? row >> 5 : 0], row & 31);
                        const int pos = __shfl_sync(0xffffffffu, own_pos[row >> 5 < kOwn ? row >> 5 : 0], row & 31);
                        return there && static_cast<unsigned int>(pre - lo) <= span && (a.window <= 0 || place > pos - a.window);
                    };
                    float tops[kOwn];
#pragma unroll
                    for (int k = 0; k < kOwn; ++k) tops[k] = kNone;
#pragma unroll 1
                    for (int q = 0; q < kHalf; q += 16) {
                        uint32_t x[16];
                        tmem_ld(t_s + q, x);
                        tmem_ld_wait(x);
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            float z = fmaf(__uint_as_float(x[k]), f, e);
                            if (masked && !sees(q + k)) z = kNone;
                            const float top = warp_max(z);
#pragma unroll
                            for (int m = 0; m < kOwn; ++m)
                                if (q + k == 32 * m + lane) tops[m] = top;
                        }
                    }
#pragma unroll
                    for (int m = 0; m < kOwn; ++m)
                        if (32 * m + lane < kHalf) room(buffer, quarter)[32 * m + lane] = tops[m];
                    if (!meet()) break;
                    float down[kOwn];
                    bool moves = false;
                    bare = false;
#pragma unroll
                    for (int m = 0; m < kOwn; ++m) {
                        down[m] = 1.f;
                        const int row = min(32 * m + lane, kHalf - 1);
                        float top = kNone;
#pragma unroll
                        for (int w = 0; w < 4; ++w) top = fmaxf(top, room(buffer, w)[row]);
                        const float old = s_ref[version][half][row];   // kOffset - reference
                        float now = old;
                        if (top > kNone && top + old > kLimit) {
                            now = kOffset - top;
                            down[m] = exp2_approx(now - old);
                            moves = true;
                        }
                        if (32 * m + lane < kHalf) {
                            s_ref[version ^ 1][half][row] = now;
                            bare = bare || now > 1e38f;
                        }
                    }
                    version ^= 1;
                    moves = __any_sync(0xffffffffu, moves);
                    bare = __any_sync(0xffffffffu, bare);
                    if (!meet()) break;   // (the room is P^T's again)
                    if (moves) {
#pragma unroll
                        for (int k = 0; k < kHalf; k += 2) {
                            const float dx = __shfl_sync(0xffffffffu, down[k >> 5], k & 31), dy = __shfl_sync(0xffffffffu, down[k >> 5], (k + 1) & 31);
                            sum2[k / 2] = mul2(sum2[k / 2], pack2(dx, dy));
                        }
                        if (j > 0) {
                            if (!wait(s_bar.o_done[(n - 1) & 1], ((n - 1) >> 1) & 1)) break;
                            fence_after();
#pragma unroll
                            for (int q = 0; q < kHalf; q += 16) {
                                uint32_t x[16];
                                tmem_ld(t_o + q, x);
                                tmem_ld_wait(x);
#pragma unroll
                                for (int k = 0; k < 16; ++k) x[k] = __float_as_uint(__uint_as_float(x[k]) * __shfl_sync(0xffffffffu, down[q >> 5], (q + k) & 31));
                                tmem_st16(t_o + q, x);
                            }
                            tmem_st_wait();
                        }
                    }
                    const bool counts = e_true >= kLeastScale;
#pragma unroll
                    for (int q = 0; q < kHalf; q += 16) {
                        uint32_t x[16];
                        tmem_ld(t_s + q, x);
                        tmem_ld_wait(x);
                        const float* const ref = s_ref[version][half] + q;
#pragma unroll
                        for (int k = 0; k < 16; k += 8) {
                            uint32_t h[4];
#pragma unroll
                            for (int m = 0; m < 8; m += 2) {
                                float p[2], w[2];
#pragma unroll
                                for (int u = 0; u < 2; ++u) {
                                    const float s = __uint_as_float(x[k + m + u]) * f, r = ref[k + m + u];
                                    const bool here = !masked || sees(q + k + m + u);
                                    w[u] = here ? exp2_approx(s + (r + (kSumOffset - kOffset))) : 0.f;
                                    p[u] = here && (counts || !(w[u] == w[u])) ? exp2_approx(s + e + r) : 0.f;
                                }
                                if (q / kChunk >= summed) sum2[(q + k + m) / 2] = add2(sum2[(q + k + m) / 2], pack2(w[0], w[1]));
                                h[m / 2] = pack_half2(p[0], p[1]);
                            }
                            *reinterpret_cast<uint4*>(p_to + (q + k) * 16) = make_uint4(h[0], h[1], h[2], h[3]);
                        }
                    }
                }
                fence_before();
                publish_smem();
                __syncwarp();
                if (lane == 0) bar_arrive(bar(s_bar.p_full[buffer]));
            }
            done += at.tiles;
            if (wait(s_bar.o_done[(done - 1) & 1], ((done - 1) >> 1) & 1)) {
                fence_after();
                // the sums of all tokens: over the lanes, then the four warps
#pragma unroll
                for (int q = 0; q < kChunks; ++q) {
                    float v[kChunk];
#pragma unroll
                    for (int k = 0; k < kChunk; k += 2) {
                        const float2 two = unpack2(sum2[(q * kChunk + k) / 2]);
                        v[k] = two.x;
                        v[k + 1] = two.y;
                    }
                    const float mine = lane_sums<kChunk>(v, lane);
                    if (lane < kChunk) room(done & 1, quarter)[q * kChunk + lane] = mine;
                }
                if (meet()) {
                    float sums[kOwn];
#pragma unroll
                    for (int m = 0; m < kOwn; ++m) {
                        const int row = min(32 * m + lane, kHalf - 1);
                        sums[m] = 0.f;
#pragma unroll
                        for (int w = 0; w < 4; ++w) sums[m] += room(done & 1, w)[row];
                    }
                    const int rows_here = min(kHalf, at.rows - at.row0 - half * kHalf);   // (or fewer than 0)
                    const bool whole = at.begins && at.ends;
                    float* const part = a.partial + (2 * c + (at.begins ? 1 : 0)) * static_cast<long>(S::kPart) + static_cast<long>(half * kHalf) * D;
                    float* const numbers = a.partial + (2 * c + (at.begins ? 1 : 0)) * static_cast<long>(S::kPart) + N * D + 2 * half * kHalf;
                    if (quarter == 0) {
#pragma unroll
                        for (int m = 0; m < kOwn; ++m) {
                            const int r = 32 * m + lane, row = at.row0 + half * kHalf + r;
                            if (r >= rows_here || r >= kHalf) continue;
                            const float c_row = kOffset - s_ref[version][half][r];
                            if (!whole) *reinterpret_cast<float2*>(numbers + 2 * r) = make_float2(c_row, sums[m]);
                            else if (a.lse) {
                                const int node = row / a.group;
                                a.lse[(at.start + node) * static_cast<long>(a.heads * a.group) + at.head * a.group + row - node * a.group] =
                                    (c_row - kSumOffset + log2f(sums[m])) * 0.6931471805599453f;
                            }
                        }
                    }
                    const int dim = token_in;   // O^T's lanes are dims
#pragma unroll
                    for (int q = 0; q < kHalf; q += 16) {
                        if (q >= rows_here) break;
                        uint32_t x[16];
                        tmem_ld(t_o + q, x);
                        tmem_ld_wait(x);
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            const float sum = __shfl_sync(0xffffffffu, sums[q >> 5], (q + k) & 31);
                            const int r = q + k, row = at.row0 + half * kHalf + r;
                            if (r >= rows_here || dim >= D) continue;
                            if (whole) {
                                const int node = row / a.group, hq = at.head * a.group + row - node * a.group;
                                a.out[(at.start + node) * a.out_stride + static_cast<long>(hq) * D + dim] =
                                    __float2half_rn(__uint_as_float(x[k]) * (131072.f / sum));   // 2^(kSumOffset - kOffset)
                            } else {
                                part[r * D + dim] = __uint_as_float(x[k]);
                            }
                        }
                    }
                    if (!whole && at.begins && warp == 0 && lane == 0) a.joins[c] = {at.last, static_cast<int>(c), at.start, at.row0, min(N, at.rows - at.row0), at.head};
                    meet();   // (the room is P^T's again)
                }
                fence_before();
            }
            done_with();
        }
    } else if (warp < kKeyWarp) {
        give_registers<kControlRegs>();
        if (warp < kScheduleWarp && elect_one()) {
            // ---- products: one thread for the scores, up to two tiles ahead, one for the values ----
            constexpr uint32_t kIdescS = instr_desc(N), kIdescO = instr_desc(N, true);
            const bool first = warp == kSWarp;
            bool go = true;
            auto until = [&](unsigned long long& b, uint32_t phase) {
                if (go && !bar_wait(smem_addr(&b), phase, flag)) {
                    go = false;
                    s_abort = 1;
                }
                return go;
            };
            const uint64_t q_desc = smem_desc(base + S::kQ, 128u, S::kRowGroup), k_desc = smem_desc(base + S::kK, 128u, S::kRowGroup);
            const uint64_t v_desc = smem_desc(base + S::kV, S::kRowGroup, 128u), p_desc = smem_desc(base + S::kP, S::kPGroup, 128u);
            uint32_t n = 0;
            while (until(s_bar.seg_full[seg_n % kSegments], (seg_n / kSegments) & 1)) {
                const int tiles = s_seg[seg_n % kSegments].tiles;
                if (tiles == 0) break;
                const uint32_t q_stage = seg_n % S::kQStages;
#pragma unroll 1
                for (int j = 0; j < tiles; ++j, ++n) {
                    const uint32_t stage = n % kStages, turn = (n / kStages) & 1, place = n & 1;
                    if (!until(first ? s_bar.k_full[stage] : s_bar.v_full[stage], turn)) break;
                    if (first) {
                        if (j == 0 && !until(s_bar.q_full[q_stage], (seg_n / S::kQStages) & 1)) break;
                        // scores of two tiles before have been read where these go
                        if (n >= 2 && !until(s_bar.p_full[place], ((n >> 1) - 1) & 1)) break;
                        fence_after();
                        const uint64_t q = q_desc + q_stage * (S::kQBytes >> 4), k = k_desc + stage * (S::kTileBytes >> 4);
#pragma unroll
                        for (int s = 0; s < D / 16; ++s) umma_ss(tmem + place * N, k + 16 * s, q + 16 * s, kIdescS, s > 0);
                        umma_commit(bar(s_bar.s_full[place]));
                        umma_commit(bar(s_bar.k_empty[stage]));
                        if (j + 1 == tiles) umma_commit(bar(s_bar.q_empty[q_stage]));
                    } else {
                        if (!until(s_bar.p_full[place], (n >> 1) & 1)) break;
                        fence_after();
                        const uint64_t v = v_desc + stage * (S::kTileBytes >> 4), p = p_desc + place * (S::kPBytes >> 4);
#pragma unroll
                        for (int s = 0; s < kTokens / 16; ++s) umma_ss(tmem + kO, v + s * (2 * S::kRowGroup >> 4), p + s * (2 * S::kPGroup >> 4), kIdescO, j > 0 || s > 0);
                        umma_commit(bar(s_bar.o_done[place]));
                        umma_commit(bar(s_bar.v_empty[stage]));
                    }
                }
                if (!go) break;
                bar_arrive(bar(s_bar.seg_empty[seg_n % kSegments]));
                ++seg_n;
            }
            // What was issued ends before the tensor memory goes: also where another warp has given up and this thread was through.
            umma_commit(bar(s_bar.done[warp - kSWarp]));
            unsigned int never = 0;
            bar_wait(bar(s_bar.done[warp - kSWarp]), 0, &never);
        }
        __syncwarp();
        if (warp == kQueryWarp) {
            // lane = (row of 8, chunk of 4)
            const bool wide = ((reinterpret_cast<uintptr_t>(a.q) | static_cast<uintptr_t>(a.q_stride * 2)) & 15) == 0;
            for (; next_segment(); done_with()) {
                const Segment& at = s_seg[seg_n % kSegments];
                const uint32_t stage = seg_n % S::kQStages;
                if (!wait(s_bar.q_empty[stage], ((seg_n / S::kQStages) & 1) ^ 1)) break;
                const int rows_here = min(N, at.rows - at.row0), live = (rows_here + 7) / 8;
                uint8_t* const dst = s_mem + S::kQ + stage * S::kQBytes + (lane & 7) * 16 + (lane >> 3) * 128;
#pragma unroll 1
                for (int g = 0; g < live; ++g) {
                    // Rows behind the last: the last again, nobody reads their results
                    const int row = min(at.row0 + 8 * g + (lane & 7), at.rows - 1);
                    const int token = row / a.group, hq = at.head * a.group + row - token * a.group;
                    const __half* const src = a.q + (at.start + token) * a.q_stride + static_cast<long>(hq) * D + 8 * (lane >> 3);
#pragma unroll
                    for (int k = 0; k < D / 32; ++k) {
                        uint8_t* const to = dst + g * S::kRowGroup + 4 * k * 128;
                        if (wide) {   // all on their way at once
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(to)), "l"(src + 32 * k) : "memory");
                        } else {
                            *reinterpret_cast<uint4*>(to) = load_halves_anywhere(src + 32 * k);
                        }
                    }
                }
                for (int g = live; g < N / 8; ++g)
                    for (int k = 0; k < D / 32; ++k) *reinterpret_cast<uint4*>(dst + g * S::kRowGroup + 4 * k * 128) = make_uint4(0u, 0u, 0u, 0u);
                asm volatile("cp.async.wait_all;" ::: "memory");
                publish_smem();
                __syncwarp();
                if (lane == 0) bar_arrive(bar(s_bar.q_full[stage]));
            }
        }
        if (warp == kScheduleWarp) {
            const long long u0 = total * c / ctas, u1 = total * (c + 1) / ctas;
            Walker<N> at;
            long long front = 0;
            int w = 0;
            while (w + 1 < kWarps && front + s_sum[w] <= u0) front += s_sum[w++];
            at.place(a, w * per, n, u0 - front, u1 - u0, lane);
            bool more = at.left > at.before;
            do {
                if (!wait(s_bar.seg_empty[seg_n % kSegments], ((seg_n / kSegments) & 1) ^ 1)) break;
                if (lane == 0) {
                    const int tiles = more ? at.run() : 0;
                    // the CTA that holds the item's last unit: the largest c' with total * c' / ctas <= that unit
                    const long long last_unit = u1 - at.left + at.before + (at.r.hi - at.tile) - 1;
                    s_seg[seg_n % kSegments] = {at.r.row, at.r.start, at.r.first(), at.r.held, at.r.rows, at.block * N, at.head, at.tile, tiles, at.tile == at.r.lo,
                                                at.tile + tiles == at.r.hi, static_cast<int>(((last_unit + 1) * ctas - 1) / total)};
                    bar_arrive(bar(s_bar.seg_full[seg_n % kSegments]));
                }
                __syncwarp();
                ++seg_n;
                if (!more) break;
                more = at.next(a, lane);
            } while (true);
        }
    } else {
        // ---- keys, values: a warp takes 16 tokens of every tile, which are in one page ----
        give_registers<kCodeRegs>();
        const bool keys = warp < kValueWarp;
        const int w = keys ? warp - kKeyWarp : warp - kValueWarp, P = a.b.page_tokens;
        const size_t block = paged_block_bytes(P, D);
        constexpr int kLoads = D / 32;   // 16-byte pieces of a lane: of rows r, r + 8, chunks c and (D = 128) c + 4
        // a tile of the share: its number, its segment, its place in it
        struct Place {
            uint32_t n, seg;
            int j, tiles;
        };
        auto step = [&](Place& at) {
            ++at.n;
            if (++at.j < at.tiles) return;
            at.j = 0;
            ++at.seg;
            at.tiles = wait(s_bar.seg_full[at.seg % kSegments], (at.seg / kSegments) & 1) ? s_seg[at.seg % kSegments].tiles : 0;
        };
        const int r = lane & 7, c4 = lane >> 3;
        int known_row = -1, known_first = -1, known = 0;   // 32 entries of a row of the tables, one per lane
        uint4 raw[kLoads];
        float2 scale = make_float2(1.f, 1.f);
        const uint4 zeros = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
        auto fetch = [&](const Place& at) {
            const Segment& seg = s_seg[at.seg % kSegments];
            const int token = (seg.tile + at.j) * kTokens + 16 * w, idx = token >> a.page_shift;
            if (token >= seg.held) {   // (behind the last page perhaps)
#pragma unroll
                for (int k = 0; k < kLoads; ++k) raw[k] = zeros;
                scale = make_float2(1.f, __uint_as_float(static_cast<unsigned int>(127 + static_cast<int>(kLeastScale)) << 23));
                return;
            }
            if (seg.row != known_row || (idx & ~31) != known_first) {
                known_row = seg.row;
                known_first = idx & ~31;
                known = known_first + lane < a.b.max_pages ? a.b.tables[static_cast<size_t>(known_row) * a.b.max_pages + known_first + lane] : 0;
            }
            const int page = __shfl_sync(0xffffffffu, known, idx & 31);
            const uint8_t* const blk = a.layer + (static_cast<size_t>(page) * a.heads + seg.head) * block;
            const uint8_t* const src = blk + (keys ? 0 : static_cast<size_t>(P) * D) + static_cast<size_t>(token & (P - 1)) * D;
#pragma unroll
            for (int k = 0; k < kLoads; ++k)
                raw[k] = *reinterpret_cast<const uint4*>(src + (r + 8 * (k & 1)) * D + 16 * (c4 + 4 * (k >> 1)));
            if (keys) scale = *reinterpret_cast<const float2*>(blk + 2 * static_cast<size_t>(P) * D);
        };
        Place now{0, 0, 0, 0};
        now.tiles = wait(s_bar.seg_full[0], 0) ? s_seg[0].tiles : 0;
        uint32_t left = 0;   // segments that this warp has given back
        if (now.tiles > 0) fetch(now);
        while (ok && now.tiles > 0) {
            const uint32_t stage = now.n % kStages, turn = (now.n / kStages) & 1, slot = now.n & (kSlots - 1);
            if (!wait(keys ? s_bar.k_empty[stage] : s_bar.v_empty[stage], turn ^ 1)) break;
            uint4 here[kLoads];
#pragma unroll
            for (int k = 0; k < kLoads; ++k) here[k] = raw[k];
            if (keys && lane == 0) s_scale[slot][w] = scale;   // (in place before the scores are)
            step(now);
            if (now.tiles > 0) fetch(now);
            uint8_t* const dst = s_mem + (keys ? S::kK : S::kV) + stage * S::kTileBytes + 2 * w * S::kRowGroup + r * 16;
#pragma unroll
            for (int k = 0; k < kLoads; ++k) {
                const int row = r + 8 * (k & 1), stored = c4 + 4 * (k >> 1), chunk = keys ? key_chunk<D>(row, stored) : value_chunk<D>(row, stored);
                const uint32_t b[4] = {here[k].x, here[k].y, here[k].z, here[k].w};
                uint32_t h[8];
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    h[2 * m] = code_halves(b[m], 0x4140);
                    h[2 * m + 1] = code_halves(b[m], 0x4342);
                }
                uint8_t* const to = dst + (k & 1) * S::kRowGroup + 2 * chunk * 128;
                *reinterpret_cast<uint4*>(to) = make_uint4(h[0], h[1], h[2], h[3]);
                *reinterpret_cast<uint4*>(to + 128) = make_uint4(h[4], h[5], h[6], h[7]);
            }
            publish_smem();
            __syncwarp();
            if (lane == 0) bar_arrive(keys ? bar(s_bar.k_full[stage]) : bar(s_bar.v_full[stage]));
            for (; left < now.seg; ++left)
                if (lane == 0) bar_arrive(bar(s_bar.seg_empty[left % kSegments]));
        }
    }
    fence_before();
    __syncthreads();
    if (tid == 0 && s_abort) raise_status(a.status, kPagedWait);
    if (warp == kSWarp) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemAll) : "memory");
    }
}

// Parts of the items that several CTAs share, in the CTAs' order: a warp per row, a lane D / 32 dims; eight parts are on their way at once.
constexpr int kJoinRows = 4;
template <int D, int N>
__global__ void __launch_bounds__(32 * kJoinRows) paged_tree_join_kernel(const __grid_constant__ PagedAttnArgs a) {
    constexpr int kPart = Shape<D, N>::kPart, kEach = D / 32, kAtOnce = 8;
    pdl_wait_release();
    const PagedJoin join = a.joins[blockIdx.x];
    const int c = blockIdx.x, lane = threadIdx.x & 31, r = blockIdx.y * kJoinRows + (threadIdx.x >> 5);
    if (join.last == 0 || r >= join.rows) return;
    const int parts = join.last - c + 1;
    float acc[kEach] = {}, top = kNone, sum = 0.f;
    for (int base = 0; base < parts; base += kAtOnce) {
        float2 ml[kAtOnce];
        float v[kAtOnce][kEach];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            const int part = min(base + k, parts - 1);
            const float* const p = a.partial + static_cast<long>(2 * (c + part) + (part == 0 ? 1 : 0)) * kPart;
            ml[k] = *reinterpret_cast<const float2*>(p + N * D + 2 * r);
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
            if (base + k >= parts) continue;
            const float to = fmaxf(top, ml[k].x);
            const float y = top == to ? 1.f : exp2_approx(top - to), x = ml[k].x == to ? 1.f : exp2_approx(ml[k].x - to);
            top = to;
            sum = fmaf(ml[k].y, x, sum * y);
#pragma unroll
            for (int d = 0; d < kEach; ++d) acc[d] = fmaf(v[k][d], x, acc[d] * y);
        }
    }
    const int row = join.first_row + r, node = row / a.group, hq = join.head * a.group + row - node * a.group;
    const float inv = 131072.f / sum;   // 2^(kSumOffset - kOffset)
    __half* const to = a.out + (join.token + node) * a.out_stride + static_cast<long>(hq) * D + kEach * lane;
#pragma unroll
    for (int d = 0; d < kEach; ++d) to[d] = __float2half_rn(acc[d] * inv);
    if (a.lse && lane == 0) a.lse[(join.token + node) * static_cast<long>(a.heads * a.group) + hq] = (top - kSumOffset + log2f(sum)) * 0.6931471805599453f;
}

template <int D, int N>
void launch_typed(PagedAttnArgs a, long max_rows, void* scratch, int sms, cudaStream_t st) {
    using S = Shape<D, N>;
    a.joins = static_cast<PagedJoin*>(scratch);
    a.partial = reinterpret_cast<float*>(static_cast<char*>(scratch) + (sms * sizeof(PagedJoin) + 255) / 256 * 256);
    static std::atomic<unsigned long long> set{0};
    static const bool registers = [] {   // (with fewer than the warps' shares add up to a warp would wait for them for ever)
        cudaFuncAttributes attr{};
        TQ_CUDA(cudaFuncGetAttributes(&attr, paged_tree_attn_kernel<D, N>));
        return attr.numRegs >= kLaunchRegs;
    }();
    TQ_REQUIRE(registers, "paged tree attention: the kernel was built with other registers than its warps share");
    allow_shared_memory(paged_tree_attn_kernel<D, N>, S::kSmem, set);
    launch_pdl_carved(paged_tree_attn_kernel<D, N>, dim3(static_cast<unsigned int>(sms)), dim3(kThreads), S::kSmem, 100, st, a);
    launch_pdl_carved(paged_tree_join_kernel<D, N>, dim3(static_cast<unsigned int>(sms), static_cast<unsigned int>((std::min<long>(N, max_rows) + kJoinRows - 1) / kJoinRows)),
                      dim3(32 * kJoinRows), 0, 100, st, a);
}

}  // namespace

void launch_paged_tree_attention(PagedAttnArgs a, int dim, long max_rows, void* scratch, int sms, cudaStream_t st) {
    const auto go = [&](auto d) {
        if (max_rows <= 32) launch_typed<d(), 32>(a, max_rows, scratch, sms, st);
        else if (max_rows <= 64) launch_typed<d(), 64>(a, max_rows, scratch, sms, st);
        else launch_typed<d(), 128>(a, max_rows, scratch, sms, st);
    };
    if (dim == 64) go(std::integral_constant<int, 64>{});
    else go(std::integral_constant<int, 128>{});
}

}  // namespace tq
