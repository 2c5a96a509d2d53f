// Attention over the paged 8-bit KV cache for many query rows of a request: prompts, chunks of them, drafts of several tokens.  The products are
// tcgen05.mma with S, P and O in tensor memory.
//
// The rows of a request and KV head (new tokens times the heads of the group, token-major) go in items of 256: two tiles of 128, whose softmaxes run
// in turn with each other's products.  The cache comes in tiles of 64 tokens.  As in tq_paged_attention.cu every CTA, one to an SM, takes an equal
// share of all (request, KV head, 256 rows, 64 tokens) units, an item's beginning and end counted as kItemUnits more, and an item that ends in
// another CTA than it begins in is added up behind.
//
//   S_t [128 x 64]   = Q_t [128 x D] (shared memory) . K [64 x D]^T (shared memory)         fp16 products, fp32 sums; two of them in turn for each t
//   P_t              = 2^(S_t f - m + 7)  fp16, over S_t's own columns of tensor memory
//   O_t [128 x D]   += P_t (tensor memory) . V (shared memory, transposed: rows are dims)
//
//   warps 0-3, 4-7   tile 0, tile 1: a thread per row reads its 64 scores once, keeps them in registers for the largest one and the weights, and
//                    writes its result
//   warps 8, 9       one lane issues the scores' products, the values'; the commit behind P_t(j) V(j) also says that O_t may be rescaled, and that
//                    the scores of two tiles on may go where P_t(j) was.  The products of the next item's first scores follow the last of this one's
//                    without a pause, while the softmax warps still write the results
//   warp 10          walks the CTA's share and tells the others, item by item, what is next (four items ahead at most)
//   warps 12-15      queries of tile 0, tile 1, of the next item as soon as the last scores of this one are there
//   warps 16-23      keys: bytes to shared memory a tile ahead, then as halves (code * 2^(e - e_max + 5), exact) to their place for the products
//   warps 24-31      values, transposed on the way; both in two groups that take every second tile
//
// Scales are powers of two: within a tile the pages' go into the halves without a rounding (but for those of pages more than 2^29 below the tile's
// largest), the tile's own goes into the exponent's factor (keys) or, as an integer, into the exponent (values: P V is kept in units of the largest
// scale that the row has seen).  The reference maximum m moves only when a score exceeds it by 2^8; weights are at most 2^15 then.  Where keys are of
// unequal strength one of a warp's 32 rows often has such a score (simulated, with norms spread by e^0.5: in 12 of 63 tiles, in 19 with 2^4), and its
// O is then read, multiplied and written back, behind the weights, so that the products before it end meanwhile: 4096 such tokens 181 us, 190 with
// 2^4, 199 with that and O in front of the weights; 175 where no row moves.
//
// What bounds it: 256 rows against 64 tokens (D = 128) take 2.7 thousand cycles.  A softmax warp is at work for 2.3 of them, waits for scores for 0.3
// and writes results for 0.2; the products alone would take 1.24 (the scores' 64 columns read 6 KB of shared memory in the 32 cycles that their
// arithmetic takes, 48 in fact), the exponentials alone 1.02, the softmax of both tiles with nothing beside it 1.17, all roles' instructions fill 54
// % of the issue slots and the tensor cores and the conversions together 75 % of shared memory's cycles.  4096 new tokens of 4 x 7 heads: 175 us,
// 0.69 PFLOP/s of the causal products, 41 % of a plain matrix product's rate.  Tried beside it, of the same prompt when it took 183: scores read
// twice in loops of 32 columns, a third less code, 191; two warps to a row's 64 scores and half as many for the conversions 195; keys and values two
// tiles ahead 185.  Tiles of 128 tokens with one set of scores and one thread for all products: 699 for 8192 tokens, 668 with these.  Part of what
// the softmax takes longer here than alone is the supply of its instructions: copies of its step in a row, alone, 771 cycles each while the code is
// below 20 KB, 933 at 37 KB, 1100 at 68 KB and 2045 at 147 KB; the roles' loops here are some 30 KB together.
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

constexpr int kRows = 128;           // query rows of a tile (MMA M)
constexpr int kPairRows = 2 * kRows; // of an item
constexpr int kTokens = 64;          // of a unit
constexpr int kMmaWarp = 8, kScheduleWarp = 10, kQueryWarp = 12, kKeyWarp = 16, kWarps = 32, kThreads = 32 * kWarps;
// Registers a thread after the warpgroups (of four warps) have split what the CTA was launched with: 1024 threads of 64.
constexpr int kSoftmaxRegs = 120, kMmaRegs = 40, kCodeRegs = 48;
static_assert(256 * kSoftmaxRegs + 256 * kMmaRegs + 512 * kCodeRegs <= kThreads * 64, "the shares are the launch's");
constexpr int kWarpTokens = 16;      // of a tile's tokens that a warp turns into halves
constexpr int kItemUnits = 4;        // what an item's beginning and end cost, in units
constexpr int kStages = 4;           // of keys and of values, as halves
constexpr int kRefs = 8;             // tiles whose scales are kept
// Weights are held times 2^7, and at most 2^15: halves that are normal numbers down to 2^-21 of the reference, and 2^-32 of it off below: of 131072
// tokens' values 2^-15 of the largest one at the very worst, 1/16 of the result's rounding.  Their sums are of the numbers before that rounding, so that
// a row with one large weight is off by that one's, 2^-11 at most: trees whose rows' largest weights are 0.4 at their median are 2.2e-4 to 2.4e-4 of
// their norm off, 2.05e-4 of which is the results' own rounding.  (With sums of the halves, simulated, 2.2e-4, for 64 conversions more to a row and
// tile.)
constexpr float kOffset = 7.f, kSlack = 8.f;
// Of a tile's values against the largest so far: a weight times 2^-60 is 0 as a half, and their sum, which is taken of these, far from it
constexpr int kLeastLower = -60;
constexpr float kHeadroom = 32.f;    // largest factor of a code in the halves
constexpr float kLeastFactor = 5.9604645e-8f;   // the least one, 2^-24: a half's last place
constexpr uint32_t kTmemAll = 512;

template <int D>
struct Shape {
    static constexpr uint32_t kRowGroup = 16 * D;          // 8 rows of queries or keys: D / 8 core matrices of 128 bytes
    // 8 dims of values, 16 core matrices; a warp's stores, 8 dims apart in pairs of lanes, would meet in the same banks without the 16
    static constexpr uint32_t kDimGroup = 16 * kTokens + 16;
    static constexpr uint32_t kQBytes = kRows / 8 * kRowGroup, kKBytes = kTokens / 8 * kRowGroup, kVBytes = D / 8 * kDimGroup;
    static constexpr uint32_t kQ = 0, kK = 2 * kQBytes, kV = kK + kStages * kKBytes, kRaw = kV + kStages * kVBytes;
    static constexpr uint32_t kRawWarp = kWarpTokens * D;   // bytes, for each of the sixteen warps that make them halves
    static constexpr uint32_t kSmem = kRaw + 16 * kRawWarp;
    static constexpr int kPart = kPairRows * (D + 2);      // floats: [D / 4][256 rows][4], then (maximum, sum) of each row
};

// A request of many rows; all lanes of a warp hold the same.
struct Request {
    int row, start, count, held, rows;
    __device__ __forceinline__ int first() const { return held - count; }
    __device__ __forceinline__ int pairs() const { return (rows + kPairRows - 1) / kPairRows; }
    // tiles of the cache that the rows of a pair see
    template <bool TREE>
    __device__ __forceinline__ void tiles(const PagedAttnArgs& a, int pair, int& lo, int& hi) const {
        // Any row may see any place.  Requests that are chains go the same way, past tiles that a causal row tile leaves out and with a look at the nodes in
        // each tile of new tokens: 4096 from an empty cache 887 us, under any window (the plain kernel: 182, and 83 with a window of 512).
        if constexpr (TREE) {
            lo = a.window > 0 ? max(0, first() - a.window + 1) / kTokens : 0;
            hi = (held - 1) / kTokens + 1;
            return;
        }
        const int last = first() + (min(rows, (pair + 1) * kPairRows) - 1) / a.group;
        hi = last / kTokens + 1;
        lo = a.window > 0 ? max(0, first() + pair * kPairRows / a.group - a.window + 1) / kTokens : 0;
    }
};
// The first request of many rows from i on (lanes look at 32 at a time); n if there is none.
template <bool TREE>
__device__ __forceinline__ int next_request(const PagedAttnArgs& a, int i, int n, int lane, Request& r) {
    for (int base = i; base < n; base += 32) {
        const int mine = min(base + lane, n - 1);
        Request x;
        x.row = a.b.rows[mine];
        x.start = a.b.starts[mine];
        x.count = a.b.starts[mine + 1] - x.start;
        x.held = a.b.held[mine];
        bool many = base + lane < n && x.count * a.group > a.few_rows;
        if constexpr (TREE) many = many && a.b.nodes[x.start].good;
        const unsigned int found = __ballot_sync(0xffffffffu, many);
        if (found) {
            const int src = __ffs(static_cast<int>(found)) - 1;
            r.row = __shfl_sync(0xffffffffu, x.row, src);
            r.start = __shfl_sync(0xffffffffu, x.start, src);
            r.count = __shfl_sync(0xffffffffu, x.count, src);
            r.held = __shfl_sync(0xffffffffu, x.held, src);
            r.rows = r.count * a.group;
            return base + src;
        }
    }
    return n;
}
// Tiles of all pairs of a request (the lanes take pairs in turn).
template <bool TREE>
__device__ __forceinline__ long long request_tiles(const PagedAttnArgs& a, const Request& r, int lane) {
    long long sum = 0;
    for (int p = lane; p < r.pairs(); p += 32) {
        int lo, hi;
        r.tiles<TREE>(a, p, lo, hi);
        sum += hi - lo + kItemUnits;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
}

// Of numbers that are not negative.  TREE: where 32 bits hold both the division is a quarter as long, and four of them are in front of a CTA's first
// product (a tree of 8 nodes over 4096 tokens: 20.7 us, 19.0 with this and what else comes sooner below).  In a prompt of 4096 tokens the same
// changes take 4 us more of 171 than they save, by where they put the other warps' code.
template <bool TREE>
__device__ __forceinline__ long long quotient(long long x, long long by) {
    if constexpr (!TREE) return x / by;
    return (x | by) >> 32 ? x / by : static_cast<long long>(static_cast<unsigned int>(x) / static_cast<unsigned int>(by));
}

// A CTA's share of the units: (request, KV head, pair, tile), the tile running fastest.
template <bool TREE>
struct Walker {
    Request r;
    int i, n, head, pair, lo, hi, tile;
    int before;          // units of kItemUnits that come in front of the present tile
    long long left;
    __device__ __forceinline__ void place(const PagedAttnArgs& a, int request, int requests, long long skip, long long units, int lane) {
        n = requests;
        left = units;
        i = next_request<TREE>(a, request, n, lane, r);
        long long sum;
        while (i < n && skip >= (sum = request_tiles<TREE>(a, r, lane)) * a.heads) {
            skip -= sum * a.heads;
            i = next_request<TREE>(a, i + 1, n, lane, r);
        }
        if (i >= n) {   // (not with a share of units that exist)
            left = 0;
            return;
        }
        head = static_cast<int>(quotient<TREE>(skip, sum));
        skip -= head * sum;
        for (int base = 0;; base += 32) {   // the pair in which the rest lies
            int l = 0, h = 0;
            if (base + lane < r.pairs()) r.template tiles<TREE>(a, base + lane, l, h);
            int upto = base + lane < r.pairs() ? h - l + kItemUnits : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int t = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += t;
            }
            const unsigned int beyond = __ballot_sync(0xffffffffu, upto > skip);
            if (beyond || base + 32 >= r.pairs()) {
                const int src = beyond ? __ffs(static_cast<int>(beyond)) - 1 : 31;
                pair = base + src;
                lo = __shfl_sync(0xffffffffu, l, src);
                hi = __shfl_sync(0xffffffffu, h, src);
                const int in = static_cast<int>(skip - (__shfl_sync(0xffffffffu, upto, src) - (hi - lo + kItemUnits)));
                before = max(0, kItemUnits - in);
                tile = lo + max(0, in - kItemUnits);
                return;
            }
            skip -= __shfl_sync(0xffffffffu, upto, 31);
        }
    }
    // Tiles of the present item that belong to the share.
    __device__ __forceinline__ int run() const { return static_cast<int>(min(static_cast<long long>(hi - tile), max(0ll, left - before))); }
    __device__ __forceinline__ bool next(const PagedAttnArgs& a, int lane) {
        left -= before + run();
        if (left <= 0) return false;
        if (++pair == r.pairs()) {
            pair = 0;
            if (++head == a.heads) {
                head = 0;
                i = next_request<TREE>(a, i + 1, n, lane, r);
                if (i >= n) return false;
            }
        }
        r.template tiles<TREE>(a, pair, lo, hi);
        tile = lo;
        before = kItemUnits;
        return left > before;
    }
};
// The part of an item that a CTA does, as the scheduling warp tells the others.
struct Segment {
    int row, start, first, held;   // of the request: row of the tables, first token, position of its first new token, tokens
    int rows, row0, head;          // its query rows, the first of this item
    int tile, tiles;               // (0: the end)
    int begins, ends;              // whether it holds the item's first and last tile
    int last;                      // the CTA in which the item ends
    __device__ __forceinline__ bool two() const { return rows - row0 > kRows; }
    // Row tiles that are at work; tiles of the cache that one takes, and the first of them
    template <bool TREE>
    __device__ __forceinline__ int teams() const { return two() || (TREE && tiles > 1) ? 2 : 1; }
    template <bool TREE>
    __device__ __forceinline__ bool split() const { return TREE && !two(); }
};
constexpr int kSegments = 4;
constexpr int kSegmentReaders = 30;   // warps: softmax, products, queries, keys, values

struct Bars {
    unsigned long long q_full[2], q_empty[2], s_full[2][2], p_full[2][2], o_done[2][2], o_empty[2], k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages], merge, seg_full[kSegments], seg_empty[kSegments], done[2];
};

// The larger of powers of two and zeros by their bits, of those that are numbers.
__device__ __forceinline__ uint32_t largest_scale(uint32_t bits) { return __reduce_max_sync(0xffffffffu, bits < 0x7f800000u ? bits : 0u); }
// A page's scale against the tile's largest, times kHeadroom: what its codes are multiplied with (0 where that is below a half's range; NaN stays).
__device__ __forceinline__ float code_factor(uint32_t bits, uint32_t largest) {
    if (bits >= 0x7f800000u) return __uint_as_float(bits);
    const int e = static_cast<int>(bits) - static_cast<int>(largest) + __float_as_int(kHeadroom);
    return bits == 0u || e <= 0 ? 0.f : __int_as_float(e);
}
// Where a chunk of a row stands in a warp's part of shared memory.
template <int D>
__device__ __forceinline__ int raw_chunk(int row, int c) {
    if constexpr (D == 128) return c ^ (row & 7);
    else return c ^ ((row >> 1) & 3);
}
// Two bytes as halves of code * factor: (1024 + b) * factor - 1152 * factor, both exact, one rounding that is none.
__device__ __forceinline__ uint32_t scaled_halves(uint32_t w, uint32_t which, __half2 factor, __half2 off) {
    const uint32_t raw = __byte_perm(w, 0x64646464u, which);
    const __half2 h = __hfma2(*reinterpret_cast<const __half2*>(&raw), factor, off);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// The columns of a tile from token tb on that hold new tokens which the row of node `number` at position pos sees, as bits (by all lanes).
__device__ __noinline__ uint64_t seen_nodes(const PagedAttnArgs& a, const Segment& at, int tb, int number, int pos, int lane) {
    uint64_t seen = 0;
#pragma unroll 1
    for (int h = 0; h < 2; ++h) {
        const int token = tb + 32 * h + lane;
        const bool there = token >= at.first && token < at.held;
        int lo = kNoNode, place = 0;
        unsigned int span = 0;
        if (there) {
            const PagedNode node = a.b.nodes[at.start + token - at.first];
            lo = node.pre;
            span = static_cast<unsigned int>(node.last - node.pre);
            place = at.first + node.depth;
        }
        const uint32_t some = __ballot_sync(0xffffffffu, there);
        uint32_t bits = 0;
#pragma unroll 1
        for (int e0 = 0; e0 < 32; e0 += 4) {   // (most tiles hold few new tokens, or none)
            if (!(some >> e0 & 0xfu)) continue;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int e = e0 + k, lo_e = __shfl_sync(0xffffffffu, lo, e), place_e = __shfl_sync(0xffffffffu, place, e);
                const unsigned int span_e = __shfl_sync(0xffffffffu, span, e);
                if (node_below(number, lo_e, span_e) && (a.window <= 0 || place_e > pos - a.window)) bits |= 1u << e;
            }
        }
        seen |= static_cast<uint64_t>(bits) << (32 * h);
    }
    return seen;
}
// The weights of a tile whose pages' values lie so far apart that their codes went into the product alone: sixteen columns of one page at a time, its
// scale against the row's unit in the exponents.  Returns their sum, without the scales.  (Out of the way: its scores come from tensor memory again.)
__device__ __noinline__ float apart_weights(uint32_t t_s, uint64_t seen, float f, float m, float4 parts, float vref) {
    float all = 0.f;
#pragma unroll 1
    for (int g = 0; g < 4; ++g) {
        const float part = g == 0 ? parts.x : g == 1 ? parts.y : g == 2 ? parts.z : parts.w;
        const float lower = part > 0.f ? static_cast<float>(max((static_cast<int>(__float_as_uint(part)) - static_cast<int>(__float_as_uint(vref))) >> 23, kLeastLower)) : 0.f;
        const float shift = m - kOffset - lower;
        uint32_t x[16], p[8];
        tmem_ld(t_s + 16 * g, x);
        tmem_ld_wait(x);
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float w = seen >> (16 * g + e) & 1 ? exp2_approx(fmaf(__uint_as_float(x[e]), f, -shift)) : 0.f;
            sum += w;
            x[e] = __float_as_uint(w);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = pack_half2(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1]));
        tmem_st(t_s + 8 * g, p);   // (columns that have been read)
        all = fmaf(sum, exp2_approx(-lower), all);
    }
    return all;
}
// 32 dims of a row of the first team, and of the second's, in their units.
__device__ __forceinline__ void add_second(uint32_t (&x)[32], uint32_t taddr, float first, float second) {
    uint32_t y[32];
    tmem_ld(taddr, y);
    tmem_ld_wait(y);
#pragma unroll
    for (int e = 0; e < 32; ++e) x[e] = __float_as_uint(fmaf(__uint_as_float(y[e]), second, __uint_as_float(x[e]) * first));
}

// TREE: trees of drafts (paged_tree_kernel in tq_paged_plan.cu numbers the nodes): a row sees the tokens in front of the new ones, its ancestors and
// itself.  A request has some tens to some hundreds of rows there, so that many items have no second row tile; its warps then take every second
// tile of the cache for the first one's rows, with a maximum, a sum and an O of their own, and the two are added up at the item's end (both read the
// same lanes of tensor memory).  16 requests of 8 to 16 nodes, 7 rows each, over 61 thousand tokens of 4 heads: 44 us replayed in a
// graph, 10 of which are one CTA's way to its first product and from its last one to the result.  Over a long cache a tile takes 1.9 thousand cycles
// with 25 rows as with 125, and 2.7 with two row tiles: for few rows the keys bound it, whose warps' way from one of their tiles to the next (every second one) is 3.7 thousand cycles: 0.5 for
// the bytes, 1.7 to make them halves, 1.1 to find the next, each instruction behind some 13 cycles of others.  Tried beside it: the
// products turned around (tokens as their 128 rows, query rows as 32, 64 or 128 columns, a softmax thread per token), which takes a tile's products as
// long as there are rows: 90 us, since each thread then keeps a sum for every row and four warps have to agree on every reference; keys and values
// from memory through registers to their place, without the bytes in shared memory, and four threads that issue products: 50; the bytes of two tiles
// on their way, with three stages of halves instead of four: 46, but a fifteenth less where a request has 16 rows.
template <int D, bool TREE>
__global__ void __launch_bounds__(kThreads, 1) paged_prompt_kernel(const __grid_constant__ PagedAttnArgs a) {
    using S = Shape<D>;
    extern __shared__ __align__(1024) uint8_t s_mem[];
    __shared__ __align__(8) Bars s_bar;
    // units of each warp's requests; later the second team's maximum, sum and unit (its exponent) of each row: there is no more room
    __shared__ __align__(16) uint8_t s_room[TREE ? 9 * kRows : kWarps * 8];
    long long* const s_sum = reinterpret_cast<long long*>(s_room);
    float* const s_top2 = reinterpret_cast<float*>(s_room);
    float* const s_sum2 = s_top2 + (TREE ? kRows : 0);
    uint8_t* const s_unit2 = s_room + (TREE ? 8 * kRows : 0);
    __shared__ float s_kref[kRefs], s_vref[kRefs];
    __shared__ __align__(16) float s_vpart[kRefs][kTokens / kWarpTokens];   // the values' scales of a tile's parts, of one page each
    __shared__ __align__(16) Segment s_seg[kSegments];
    __shared__ uint32_t s_tmem;
    __shared__ unsigned int s_abort;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    auto bar = [&](unsigned long long& b) { return smem_addr(&b); };
    if (tid == 0) {
        for (int k = 0; k < 2; ++k) {
            bar_init(bar(s_bar.q_full[k]), 2);
            bar_init(bar(s_bar.q_empty[k]), 1);
            for (int b = 0; b < 2; ++b) {
                bar_init(bar(s_bar.s_full[k][b]), 1);
                bar_init(bar(s_bar.p_full[k][b]), 4);
                bar_init(bar(s_bar.o_done[k][b]), 1);
            }
            bar_init(bar(s_bar.o_empty[k]), 4);
            bar_init(bar(s_bar.done[k]), 1);
        }
        for (int k = 0; k < kStages; ++k) {
            bar_init(bar(s_bar.k_full[k]), 4);
            bar_init(bar(s_bar.k_empty[k]), 1);
            bar_init(bar(s_bar.v_full[k]), 4);
            bar_init(bar(s_bar.v_empty[k]), 1);
        }
        bar_init(bar(s_bar.merge), 4);
        for (int k = 0; k < kSegments; ++k) {
            bar_init(bar(s_bar.seg_full[k]), 1);
            bar_init(bar(s_bar.seg_empty[k]), kSegmentReaders);
        }
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    auto allocate = [&]() {
        if (warp != kMmaWarp) return;
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)), "r"(kTmemAll) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        fence_before();
    };
    // (in front of the wait for the kernel before: nobody beside this CTA can be in want of tensor memory meanwhile, since its threads have all of the
    // SM's registers)
    static_assert(kThreads * 64 == 65536);
    if constexpr (TREE) allocate();
    pdl_wait_release();
    int n = planned(a.b.header, a.sizes, a.status).requests;
    if constexpr (TREE) {
        if (n > 0 && a.b.header->state != kPagedTree) {   // (a plan of the same sizes that has no trees)
            if (blockIdx.x == 0 && tid == 0) raise_status(a.status, kPagedOtherPlan);
            n = 0;
        }
    }
    const int per = (n + kWarps - 1) / kWarps;
    {
        const int end = min(n, (warp + 1) * per);
        long long mine = 0;
        Request r;
        for (int i = next_request<TREE>(a, warp * per, end, lane, r); i < end; i = next_request<TREE>(a, i + 1, end, lane, r)) mine += request_tiles<TREE>(a, r, lane) * a.heads;
        if (lane == 0) s_sum[warp] = mine;
    }
    __syncthreads();
    static_assert(kWarps == 32, "a lane for each warp's units");
    long long total = 0, upto = 0;   // (TREE) units of the warps up to the lane's
    if constexpr (TREE) {
        upto = s_sum[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long t = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += t;
        }
        total = __shfl_sync(0xffffffffu, upto, 31);
    } else {
#pragma unroll
        for (int k = 0; k < kWarps; ++k) total += s_sum[k];
    }
    const long long ctas = min(static_cast<long long>(gridDim.x), total), c = blockIdx.x;
    if (tid == 0) a.joins[c].last = 0;
    if (c >= ctas) {
        if (TREE && warp == kMmaWarp) {
            fence_after();
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(s_tmem), "r"(kTmemAll) : "memory");
        }
        return;
    }
    if constexpr (!TREE) allocate();
    __syncthreads();   // (TREE: every warp has read the sums, in whose place the second team's will be)
    fence_after();
    const uint32_t tmem = s_tmem;
    const uint32_t base = smem_addr(s_mem);
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

    if (warp < kMmaWarp) {
        // ---- softmax: a thread per row ----
        take_registers<kSoftmaxRegs>();
        const int t = warp >> 2, r_in = tid & (kRows - 1);
        const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;   // this warp's 32 lanes of tensor memory
        const uint32_t t_s0 = tmem + lanes + t * 2 * kTokens, t_o = tmem + lanes + 4 * kTokens + t * D;
        const bool out_wide = ((reinterpret_cast<uintptr_t>(a.out) | static_cast<uintptr_t>(a.out_stride * 2)) & 15) == 0;
        uint32_t done = 0, count = 0;   // tiles of this thread's so far, and of the share (their scales' place)
        uint32_t merged = 0;            // items that two teams shared
        while (next_segment()) {
            const Segment& at = s_seg[seg_n % kSegments];
            const int tiles = at.tiles, tile0 = at.tile;
            if (t < at.teams<TREE>()) {
                const bool split = at.split<TREE>();
                const int row = at.row0 + (split ? 0 : t * kRows) + r_in, in_row = min(row, at.rows - 1);
                const int token = at.start + in_row / a.group, hq = at.head * a.group + in_row % a.group;
                int pos = at.first + in_row / a.group, number = 0;   // (TREE: by the node's depth; its number)
                if constexpr (TREE) {
                    const PagedNode node = a.b.nodes[token];
                    pos = at.first + node.depth;
                    number = node.pre;
                }
                const bool live = row < at.rows;
                const int oldest = a.window > 0 ? max(0, pos - a.window + 1) : 0;
                // A warp without rows: it keeps the others' count (16 requests of 35 rows: 48 us, 56 with the softmax of what is not there)
                const bool idle = at.row0 + (split ? 0 : t * kRows) + 32 * (warp & 3) >= at.rows;
                // O is in units of vref: the largest of the values' scales that the row has seen (vseen), or the tile's where it sees only part of
                // the tile and the rest is larger.  It comes down again behind such a tile: a window that begins there has all its other tokens in
                // front.
                float m = -INFINITY, l = 0.f, vref = 0.f, vseen = 0.f;
                const int step = split ? 2 : 1, j0 = split ? t : 0;
                uint32_t n = done;
                for (int j = j0; j < tiles; j += step, ++n) {
                    const uint32_t ref = (count + j) & (kRefs - 1);
                    if (!wait(s_bar.s_full[t][n & 1], (n >> 1) & 1)) break;
                    if (idle) {
                        if (lane == 0) bar_arrive(bar(s_bar.p_full[t][n & 1]));
                        continue;
                    }
                    fence_after();
                    const uint32_t t_s = t_s0 + (n & 1) * kTokens;
                    uint32_t x[32], y[32];
                    const float kref = s_kref[ref], vref_here = TREE ? fabsf(s_vref[ref]) : s_vref[ref];
                    const bool apart = TREE && s_vref[ref] < 0.f;   // the codes are there alone
                    tmem_ld(t_s, x);
                    tmem_ld(t_s + 32, y);
                    const int tb = (tile0 + j) * kTokens;
                    const float f = fmaxf(kref * a.scale_log2, 1.1754944e-38f);   // (not 0: minus infinity times it)
                    // columns eldest .. newest are seen (TREE: and new tokens by their nodes)
                    const int newest = (TREE ? at.first - 1 : pos) - tb, eldest = oldest - tb;
                    float vt = TREE || (newest >= 0 && eldest < kTokens) ? vref_here : 0.f, vpart = vt;   // (what a row does not see leaves its unit alone)
                    uint64_t all_seen = ~0ull;   // (TREE)
                    tmem_ld_wait(x);
                    tmem_ld_wait(y);
                    if (__any_sync(0xffffffffu, newest < kTokens - 1 || eldest > 0)) {
                        // a bit for each column
                        uint64_t seen = (newest >= 63 ? ~0ull : newest < 0 ? 0ull : (2ull << newest) - 1) & (eldest <= 0 ? ~0ull : eldest > 63 ? 0ull : ~0ull << eldest);
                        if constexpr (TREE) seen |= seen_nodes(a, at, tb, number, pos, lane);
                        const uint32_t lo = static_cast<uint32_t>(seen), hi = static_cast<uint32_t>(seen >> 32);
                        if constexpr (TREE) all_seen = seen;
                        const float4 parts = *reinterpret_cast<const float4*>(s_vpart[ref]);
                        vpart = fmaxf(fmaxf(lo & 0xffffu ? parts.x : 0.f, lo >> 16 ? parts.y : 0.f), fmaxf(hi & 0xffffu ? parts.z : 0.f, hi >> 16 ? parts.w : 0.f));
                        if (code_factor(__float_as_uint(vpart), __float_as_uint(vt)) < kLeastFactor) vt = 0.f;   // (all that it sees counts as 0)
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            if (!(lo >> e & 1)) x[e] = 0xff800000u;   // (minus infinity, times f)
                            if (!(hi >> e & 1)) y[e] = 0xff800000u;
                        }
                    }
                    float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int e = 0; e < 32; ++e) tops[e & 3] = fmaxf(fmaxf(tops[e & 3], __uint_as_float(x[e])), __uint_as_float(y[e]));
                    float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
                    top *= f;   // (f is positive; NaN columns do not count)
                    float4 parts = make_float4(0.f, 0.f, 0.f, 0.f);   // (apart) the scales of what the row sees, sixteen columns each
                    if (apart) {
                        parts = *reinterpret_cast<const float4*>(s_vpart[ref]);
                        parts.x = all_seen & 0xffffu ? parts.x : 0.f;
                        parts.y = all_seen & 0xffff0000u ? parts.y : 0.f;
                        parts.z = all_seen & 0xffff00000000u ? parts.z : 0.f;
                        parts.w = all_seen >> 48 ? parts.w : 0.f;
                        vt = vpart = fmaxf(fmaxf(parts.x, parts.y), fmaxf(parts.z, parts.w));
                    }
                    const bool jump = top > m + kSlack || (m == -INFINITY && top > m);
                    float both = 1.f;
                    vseen = fmaxf(vseen, vpart);
                    const float vnew = fmaxf(vseen, vt);
                    const bool moves = __any_sync(0xffffffffu, jump || vnew != vref);
                    if (moves) {
                        const float to = jump ? top : m;
                        const float down = jump ? (m == -INFINITY ? 0.f : exp2_approx(m - to)) : 1.f;
                        both = vnew > 0.f ? down * (vref / vnew) : 0.f;
                        l *= down;
                        m = to;
                        vref = vnew;
                    }
                    // the values' scale against the largest so far, as a whole number in the exponent
                    const float lower = vt > 0.f ? static_cast<float>(max((static_cast<int>(__float_as_uint(vt)) - static_cast<int>(__float_as_uint(vref))) >> 23, kLeastLower)) : 0.f;
                    const float shift = (m == -INFINITY ? 0.f : m) - kOffset - lower;
                    const unsigned long long f2 = pack2(f, f), shift2 = pack2(-shift, -shift);
                    unsigned long long sums[2] = {0ull, 0ull};
                    auto weights = [&](const uint32_t (&v)[32], uint32_t to) {
                        uint32_t p[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            float2 w = unpack2(fma2(pack2(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])), f2, shift2));
                            w.x = exp2_approx(w.x);
                            w.y = exp2_approx(w.y);
                            sums[e & 1] = add2(sums[e & 1], pack2(w.x, w.y));
                            p[e] = pack_half2(w.x, w.y);
                        }
                        tmem_st16(to, p);
                    };
                    if (apart) {
                        l += apart_weights(t_s, all_seen, f, m == -INFINITY ? 0.f : m, parts, vref);
                    } else {
                        weights(x, t_s);
                        weights(y, t_s + 16);
                        const float2 both_sums = unpack2(add2(sums[0], sums[1]));
                        const float sum = both_sums.x + both_sums.y;
                        l = fmaf(sum, exp2_approx(-lower), l);
                    }
                    if (moves && j > j0) {   // O to the new reference: behind the weights, which take as long as the products that it waits for
                        if (!wait(s_bar.o_done[t][(n - 1) & 1], ((n - 1) >> 1) & 1)) break;
                        fence_after();
#pragma unroll 1
                        for (int q = 0; q < D; q += 32) {
                            tmem_ld(t_o + q, x);
                            tmem_ld_wait(x);
#pragma unroll
                            for (int e = 0; e < 32; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * both);
                            tmem_st(t_o + q, x);
                        }
                    }
                    tmem_st_wait();
                    fence_before();
                    __syncwarp();
                    if (lane == 0) bar_arrive(bar(s_bar.p_full[t][n & 1]));
                }
                done += (tiles - j0 + step - 1) / step;
                bool last = wait(s_bar.o_done[t][(done - 1) & 1], ((done - 1) >> 1) & 1);
                const bool shared = split && tiles > 1;
                float second = 0.f;   // the second team's unit, against this one's reference
                if constexpr (TREE) {
                    if (last && shared) {
                        if (t == 1) {
                            s_top2[r_in] = m;
                            s_sum2[r_in] = l;
                            s_unit2[r_in] = static_cast<uint8_t>(__float_as_uint(vref) >> 23);
                            fence_before();
                            __syncwarp();
                            if (lane == 0) bar_arrive(bar(s_bar.merge));
                            last = false;   // (the first team does the rest)
                        } else {
                            last = wait(s_bar.merge, merged++ & 1);
                            const float m1 = s_top2[r_in], top = fmaxf(m, m1);
                            const float x0 = m == top || m == -INFINITY ? 1.f : exp2_approx(m - top), x1 = m1 == top || m1 == -INFINITY ? 1.f : exp2_approx(m1 - top);
                            l = fmaf(l, x0, s_sum2[r_in] * x1);
                            vref *= x0;
                            second = __uint_as_float(static_cast<uint32_t>(s_unit2[r_in]) << 23) * x1 * (1.f / kHeadroom);
                            m = top;
                        }
                    }
                }
                if (last) {
                    fence_after();
                    const bool begins = at.begins, ends = at.ends;
                    float unit = vref * (1.f / kHeadroom), one = unit;
                    if (shared) unit = 1.f;
                    uint32_t x[32];
                    if (begins && ends) {
                        const float inv = unit / l;
                        __half* const dst = a.out + token * a.out_stride + static_cast<long>(hq) * D;
#pragma unroll 1
                        for (int q = 0; q < (TREE && idle ? 0 : D / 32); ++q) {
                            tmem_ld(t_o + 32 * q, x);
                            tmem_ld_wait(x);
                            if constexpr (TREE) {
                                if (shared) add_second(x, t_o + D + 32 * q, one, second);
                            }
                            if (!live) continue;
#pragma unroll
                            for (int e = 0; e < 32; e += 8) {
                                float v[8];
#pragma unroll
                                for (int k = 0; k < 8; ++k) v[k] = __uint_as_float(x[e + k]) * inv;
                                if (out_wide) *reinterpret_cast<uint4*>(dst + 32 * q + e) = pack_halves(v);
                                else store_halves_anywhere(dst + 32 * q + e, pack_halves(v));
                            }
                        }
                        if (live && a.lse) a.lse[token * static_cast<long>(a.heads * a.group) + hq] = (m - kOffset + log2f(l)) * 0.6931471805599453f;
                    } else {
                        float* const part = a.partial + (2 * c + (begins ? 1 : 0)) * static_cast<long>(S::kPart);
                        const int pr = t * kRows + r_in;
#pragma unroll 1
                        for (int q = 0; q < (TREE && idle ? 0 : D / 32); ++q) {
                            tmem_ld(t_o + 32 * q, x);
                            tmem_ld_wait(x);
                            if constexpr (TREE) {
                                if (shared) add_second(x, t_o + D + 32 * q, one, second);
                            }
#pragma unroll
                            for (int e = 0; e < 32; e += 4)
                                *reinterpret_cast<float4*>(part + ((8 * q + e / 4) * kPairRows + pr) * 4) =
                                    make_float4(__uint_as_float(x[e]) * unit, __uint_as_float(x[e + 1]) * unit, __uint_as_float(x[e + 2]) * unit, __uint_as_float(x[e + 3]) * unit);
                        }
                        *reinterpret_cast<float2*>(part + kPairRows * D + 2 * pr) = make_float2(m, l);
                        if (begins && t == 0 && r_in == 0) {
                            a.joins[c] = {at.last, static_cast<int>(c), at.start, at.row0, min(kPairRows, at.rows - at.row0), at.head};
                        }
                    }
                    fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        bar_arrive(bar(s_bar.o_empty[t]));
                        if (TREE && shared) bar_arrive(bar(s_bar.o_empty[1]));
                    }
                }
            }
            count += tiles;
            done_with();
        }
    } else if (warp < kKeyWarp) {
        // ---- products ----
        give_registers<kMmaRegs>();
        constexpr uint32_t kIdescS = instr_desc(kTokens), kIdescO = instr_desc(D);
        if (warp < kScheduleWarp && elect_one()) {
            // One thread for the scores, up to two tiles of the cache ahead, one for P V: a commit holds its thread up until the products in front
            // are done, and what comes between it and the next product is beside the other thread's products then.  (One thread for all: 3.7 thousand
            // cycles for 128 tokens with nothing else to do, of which the products take 2.1; one for each row tile, with 35 rows in one tile: 2.7
            // thousand cycles for 64 tokens.)
            const bool first = warp == kMmaWarp;
            bool go = true;
            auto until = [&](unsigned long long& b, uint32_t phase) {
                if (go && !bar_wait(smem_addr(&b), phase, flag)) {
                    go = false;
                    s_abort = 1;
                }
                return go;
            };
            const uint64_t q_desc = smem_desc(base + S::kQ, S::kRowGroup), k_desc = smem_desc(base + S::kK, S::kRowGroup), v_desc = smem_desc(base + S::kV, S::kDimGroup);
            // Tiles of the cache; items of each row tile (a bit each, the parity); scores, or P V, of each row tile
            uint32_t turns = 0, items = 0, n0 = 0, n1 = 0;
            while (until(s_bar.seg_full[seg_n % kSegments], (seg_n / kSegments) & 1)) {
                const int tiles = s_seg[seg_n % kSegments].tiles, pair = s_seg[seg_n % kSegments].two() ? 2 : 1;
                if (tiles == 0) break;
                const bool split = s_seg[seg_n % kSegments].split<TREE>();   // (row tile t takes the tiles t, t + 2, ... with the first one's queries)
#pragma unroll 1
                for (int j = 0; j < tiles; ++j, ++turns) {
                    const uint32_t stage = turns % kStages, turn = (turns / kStages) & 1;
                    if (!until(first ? s_bar.k_full[stage] : s_bar.v_full[stage], turn)) break;
#pragma unroll 1
                    for (int t = split ? j & 1 : 0; t < (split ? (j & 1) + 1 : pair); ++t) {
                        const uint32_t nt = t ? n1 : n0, place = nt & 1, t_s = tmem + (2 * t + place) * kTokens;
                        if (first) {
                            if (j == 0 && !until(s_bar.q_full[split ? 0 : t], (items >> t) & 1)) break;
                            // P of two tiles before was where these scores go
                            if (nt >= 2 && !until(s_bar.o_done[t][place], ((nt >> 1) - 1) & 1)) break;
                            fence_after();
                            const uint64_t q = q_desc + (split ? 0 : t) * (S::kQBytes >> 4), k = k_desc + stage * (S::kKBytes >> 4);
#pragma unroll
                            for (int s = 0; s < D / 16; ++s) umma_ss(t_s, q + 16 * s, k + 16 * s, kIdescS, s > 0);
                            umma_commit(bar(s_bar.s_full[t][place]));
                            if (j + 1 == tiles) umma_commit(bar(s_bar.q_empty[split ? 0 : t]));
                        } else {
                            const bool begins = j == (split ? t : 0);
                            if (begins && !until(s_bar.o_empty[t], ((items >> t) & 1) ^ 1)) break;
                            if (!until(s_bar.p_full[t][place], (nt >> 1) & 1)) break;
                            fence_after();
                            const uint64_t v = v_desc + stage * (S::kVBytes >> 4);
#pragma unroll
                            for (int s = 0; s < kTokens / 16; ++s) umma_ts(tmem + 4 * kTokens + t * D, t_s + 8 * s, v + 16 * s, kIdescO, !begins || s > 0);
                            umma_commit(bar(s_bar.o_done[t][place]));
                        }
                        if (t) ++n1; else ++n0;
                    }
                    if (!go) break;
                    umma_commit(bar(first ? s_bar.k_empty[stage] : s_bar.v_empty[stage]));
                }
                items ^= pair == 2 || (!first && split && tiles > 1) ? 3u : 1u;
                bar_arrive(bar(s_bar.seg_empty[seg_n % kSegments]));
                ++seg_n;
            }
            // What was issued ends before the tensor memory goes: also where another warp has given up and this thread was through.
            umma_commit(bar(s_bar.done[warp - kMmaWarp]));
            unsigned int never = 0;
            bar_wait(bar(s_bar.done[warp - kMmaWarp]), 0, &never);
        }
        __syncwarp();
        if (warp >= kQueryWarp) {
            // lane = (row of 8, chunk of 4)
            const int t = (warp - kQueryWarp) >> 1, part = warp & 1;
            const bool wide = ((reinterpret_cast<uintptr_t>(a.q) | static_cast<uintptr_t>(a.q_stride * 2)) & 15) == 0;
            uint32_t q_n = 0;
            for (; next_segment(); done_with()) {
                const Segment& at = s_seg[seg_n % kSegments];
                if (t == 1 && !at.two()) continue;
                if (!wait(s_bar.q_empty[t], (q_n++ & 1) ^ 1)) break;
                // Rows behind the last: zeros beside live ones of a softmax warp, what is there for warps without.  (With the last row in their place
                // 148 CTAs asked the same place of the L2 cache for it a hundred times each, 20 us for a request of 35 rows.)
                const int rows_here = min(kRows, at.rows - at.row0 - t * kRows), live = (rows_here + 7) / 8, groups = (rows_here + 31) / 32 * 4;
                uint8_t* const dst = s_mem + S::kQ + t * S::kQBytes + (lane & 7) * 16 + (lane >> 3) * 128;
#pragma unroll 1
                for (int g = part; g < live; g += 2) {
                    // Rows behind the last: the last again, nobody reads their results
                    const int row = min(at.row0 + t * kRows + 8 * g + (lane & 7), at.rows - 1);
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
                for (int g = live + ((live ^ part) & 1); g < groups; g += 2)
                    for (int k = 0; k < D / 32; ++k) *reinterpret_cast<uint4*>(dst + g * S::kRowGroup + 4 * k * 128) = make_uint4(0u, 0u, 0u, 0u);
                asm volatile("cp.async.wait_all;" ::: "memory");
                publish_smem();
                __syncwarp();
                if (lane == 0) bar_arrive(bar(s_bar.q_full[t]));
            }
        }
        if (warp == kScheduleWarp) {
            const long long u0 = quotient<TREE>(total * c, ctas), u1 = quotient<TREE>(total * (c + 1), ctas);
            Walker<TREE> at;
            long long front = 0;
            int w = 0;
            if constexpr (TREE) {
                w = __ffs(static_cast<int>(__ballot_sync(0xffffffffu, upto > u0))) - 1;   // (u0 is below the total)
                if (w > 0) front = __shfl_sync(0xffffffffu, upto, w - 1);
            } else {
                while (w + 1 < kWarps && front + s_sum[w] <= u0) front += s_sum[w++];
            }
            at.place(a, w * per, n, u0 - front, u1 - u0, lane);
            bool more = at.left > at.before;
            do {
                if (!wait(s_bar.seg_empty[seg_n % kSegments], ((seg_n / kSegments) & 1) ^ 1)) break;
                if (lane == 0) {
                    const int tiles = more ? at.run() : 0;
                    // the CTA that holds the item's last unit: the largest c' with total * c' / ctas <= that unit
                    const long long last_unit = u1 - at.left + at.before + (at.hi - at.tile) - 1;
                    s_seg[seg_n % kSegments] = {at.r.row, at.r.start, at.r.first(), at.r.held, at.r.rows, at.pair * kPairRows, at.head, at.tile, tiles, at.tile == at.lo,
                                                at.tile + tiles == at.hi, static_cast<int>(quotient<TREE>((last_unit + 1) * ctas - 1, total))};
                    bar_arrive(bar(s_bar.seg_full[seg_n % kSegments]));
                }
                __syncwarp();
                ++seg_n;
                if (!more) break;
                more = at.next(a, lane);
            } while (true);
        }
    } else {
        // ---- keys, values: a warp takes 16 tokens, which are in one page, of every second tile ----
        give_registers<kCodeRegs>();
        const int role = warp - kKeyWarp, w = role & 3, P = a.b.page_tokens;
        const bool keys = role < 8;
        uint8_t* const raw = s_mem + S::kRaw + role * S::kRawWarp;
        const size_t block = paged_block_bytes(P, D);
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
        int known_row = -1, known_first = -1, known = 0;   // 32 entries of a row of the tables, one per lane
        uint2 scales = make_uint2(0u, 0u);                 // of the fetched tile's pages, one per lane, as bits
        // The 16 tokens' bytes on their way to this warp's part of shared memory, in an order in which eight rows' reads of a chunk meet in no bank.
        // (Tokens behind the request's last are read all the same, from its last page: their bytes are finite whatever was there, and no row sees
        // them.)
        auto fetch = [&](const Place& at) {
            const Segment& seg = s_seg[at.seg % kSegments];
            const int token = (seg.tile + at.j) * kTokens, first = token >> a.page_shift, pages = (min(kTokens, seg.held - token) + P - 1) >> a.page_shift;
            if (seg.row != known_row || (first & ~31) != known_first) {
                known_row = seg.row;
                known_first = first & ~31;
                known = known_first + lane < a.b.max_pages ? a.b.tables[static_cast<size_t>(known_row) * a.b.max_pages + known_first + lane] : 0;
            }
            const int page = __shfl_sync(0xffffffffu, known, (first + lane) & 31);
            scales = make_uint2(0u, 0u);
            if (lane < pages)
                scales = *reinterpret_cast<const uint2*>(a.layer + (static_cast<size_t>(page) * a.heads + seg.head) * block + 2 * static_cast<size_t>(P) * D);
            const int mine = __shfl_sync(0xffffffffu, page, min(kWarpTokens * w >> a.page_shift, pages - 1));
            const uint8_t* const src = a.layer + (static_cast<size_t>(mine) * a.heads + seg.head) * block + (keys ? 0 : static_cast<size_t>(P) * D) +
                                       static_cast<size_t>((token + kWarpTokens * w) & (P - 1)) * D + 16 * lane;
            constexpr int kChunks = D / 16, kRowsAtOnce = 32 / kChunks;
#pragma unroll
            for (int i = 0; i < kWarpTokens / kRowsAtOnce; ++i) {
                const int r = lane / kChunks + i * kRowsAtOnce;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(raw + r * D + 16 * raw_chunk<D>(r, lane % kChunks))), "l"(src + 512 * i) : "memory");
            }
        };
        // `now` is made halves of, `next`, two tiles on, is on its way
        Place now{0, 0, 0, 0};
        now.tiles = wait(s_bar.seg_full[0], 0) ? s_seg[0].tiles : 0;
        uint32_t left = 0;   // segments that this warp has given back
        if (now.tiles > 0 && (role & 4)) step(now);
        if (now.tiles > 0) fetch(now);
        while (ok && now.tiles > 0) {
            const uint2 here = scales;
            const uint32_t stage = now.n % kStages, turn = (now.n / kStages) & 1;
            const int seg_tokens = s_seg[now.seg % kSegments].held - (s_seg[now.seg % kSegments].tile + now.j) * kTokens;
            const int page = min(kWarpTokens * w >> a.page_shift, ((min(kTokens, seg_tokens) + P - 1) >> a.page_shift) - 1);
            asm volatile("cp.async.wait_all;" ::: "memory");
            __syncwarp();
            if (!wait(keys ? s_bar.k_empty[stage] : s_bar.v_empty[stage], turn ^ 1)) break;
            // a page whose values are not numbers is one whose keys are not: its tokens' columns become NaN
            const uint32_t key_bits = here.y < 0x7f800000u ? here.x : 0x7fc00000u, value_bits = here.y < 0x7f800000u ? here.y : 0u;
            const uint32_t value_ref = largest_scale(value_bits);
            // (TREE) Pages whose values would not be exact in the largest one's unit, which may be one that hardly any row sees: the codes go there alone, and
            // the weights have the scales.
            const bool apart = TREE && __any_sync(0xffffffffu, value_bits != 0u && code_factor(value_bits, value_ref) < kLeastFactor);
            if (keys) {
                // lane = (row of 8, chunk of 4)
                const uint32_t ref = largest_scale(key_bits);
                const __half2 fa = __float2half2_rn(code_factor(__shfl_sync(0xffffffffu, key_bits, page), ref)), off = __hmul2(fa, __float2half2_rn(-1152.f));
                uint8_t* const dst = s_mem + S::kK + stage * S::kKBytes + 2 * w * S::kRowGroup + (lane & 7) * 16;
#pragma unroll(TREE ? 2 : 1)
                for (int s = 0; s < D / 32; ++s) {
                    const int r = 8 * (s & 1) + (lane & 7), c0 = (lane >> 3) + 2 * (s & 2);
                    const uint4 b4 = *reinterpret_cast<const uint4*>(raw + r * D + 16 * raw_chunk<D>(r, key_chunk<D>(r, c0)));
                    const uint32_t b[4] = {b4.x, b4.y, b4.z, b4.w};
                    uint32_t h[8];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        h[2 * k] = scaled_halves(b[k], 0x4140, fa, off);
                        h[2 * k + 1] = scaled_halves(b[k], 0x4342, fa, off);
                    }
                    uint8_t* const to = dst + (s & 1) * S::kRowGroup + 2 * c0 * 128;
                    *reinterpret_cast<uint4*>(to) = make_uint4(h[0], h[1], h[2], h[3]);
                    *reinterpret_cast<uint4*>(to + 128) = make_uint4(h[4], h[5], h[6], h[7]);
                }
                if (w == 0) {   // (in place before the scores are)
                    const uint32_t part = __shfl_sync(0xffffffffu, value_bits, min(kWarpTokens * (lane & 3) >> a.page_shift, ((min(kTokens, seg_tokens) + P - 1) >> a.page_shift) - 1));
                    if (lane < kTokens / kWarpTokens) s_vpart[now.n & (kRefs - 1)][lane] = __uint_as_float(part);
                    if (lane == 0) {
                        s_kref[now.n & (kRefs - 1)] = ref > 0u ? __uint_as_float(ref) * (1.f / kHeadroom) : 1.f;
                        s_vref[now.n & (kRefs - 1)] = apart ? -__uint_as_float(value_ref) : __uint_as_float(value_ref);
                    }
                }
            } else {
                // a lane takes four dims of eight tokens
                constexpr int kLanes = D / 4, kGroups = 32 / kLanes;   // groups of 8 tokens side by side in a warp
                const int d4 = lane % kLanes;
                const __half2 fa = __float2half2_rn(apart ? kHeadroom : code_factor(__shfl_sync(0xffffffffu, value_bits, page), value_ref)), off = __hmul2(fa, __float2half2_rn(-1152.f));
                uint8_t* const dst = s_mem + S::kV + stage * S::kVBytes + (d4 >> 1) * S::kDimGroup + (d4 & 1) * 64 + 2 * w * 128;
#pragma unroll 1
                for (int s = 0; s < 2; s += kGroups) {
                    const int mine8 = s + lane / kLanes;
                    uint32_t pair[4][2];   // bytes of two tokens side by side: dims 0, 1 and 2, 3
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint32_t b[2];
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const int r = 8 * mine8 + 2 * e + k;
                            b[k] = *reinterpret_cast<const uint32_t*>(raw + r * D + 16 * raw_chunk<D>(r, value_chunk<D>(r, d4 >> 2)) + 4 * (d4 & 3));
                        }
                        pair[e][0] = __byte_perm(b[0], b[1], 0x5140);
                        pair[e][1] = __byte_perm(b[0], b[1], 0x7362);
                    }
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        const uint32_t which = (d & 1) ? 0x4342 : 0x4140;
                        uint32_t h[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) h[e] = scaled_halves(pair[e][d >> 1], which, fa, off);
                        *reinterpret_cast<uint4*>(dst + mine8 * 128 + d * 16) = make_uint4(h[0], h[1], h[2], h[3]);
                    }
                }
            }
            publish_smem();
            __syncwarp();
            if (lane == 0) bar_arrive(keys ? bar(s_bar.k_full[stage]) : bar(s_bar.v_full[stage]));
            if (TREE && now.j + 2 < now.tiles) {   // (in the same segment, as nearly always)
                now.n += 2;
                now.j += 2;
            } else {
                step(now);
                if (now.tiles > 0) step(now);
            }
            if (now.tiles > 0) fetch(now);
            for (; left < now.seg; ++left)
                if (lane == 0) bar_arrive(bar(s_bar.seg_empty[left % kSegments]));
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    if (tid == 0 && s_abort) raise_status(a.status, kPagedWait);
    if (warp == kMmaWarp) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemAll) : "memory");
    }
}

// Parts of the items that several CTAs share, in the CTAs' order: a thread takes four dims of ROWS rows, eight rows apart.  Bound by the latency of
// its loads (entry, parts, one behind the other), so what a thread reads is on its way at once: two parts of four rows where items are full (a
// prompt, 148 items of two parts, 38 MB: 7 us less than a row at a time), eight parts of a row where they are not (few rows over a long cache, cut
// into many).
constexpr int kJoinRows = 8;
template <int D, int ROWS>
__global__ void __launch_bounds__(kJoinRows * D / 4) paged_prompt_join_kernel(const __grid_constant__ PagedAttnArgs a) {
    constexpr int kPart = Shape<D>::kPart;
    pdl_wait_release();
    const PagedJoin join = a.joins[blockIdx.x];
    const int c = blockIdx.x, r0 = blockIdx.y * (kJoinRows * ROWS) + threadIdx.x % kJoinRows, d4 = threadIdx.x / kJoinRows;
    if (join.last == 0 || r0 >= join.rows) return;
    const int parts = join.last - c + 1;
    auto part_of = [&](int k) { return a.partial + (2 * (c + k) + (k == 0 ? 1 : 0)) * static_cast<long>(kPart); };
    struct Sum {
        float top, sum;
        float4 acc;
        __device__ __forceinline__ void add(float2 ml, float4 v) {
            const float to = fmaxf(top, ml.x);
            const float x = top == to || top == -INFINITY ? 1.f : exp2_approx(top - to), y = ml.x == to || ml.x == -INFINITY ? 1.f : exp2_approx(ml.x - to);
            top = to;
            sum = sum * x + ml.y * y;
            acc.x = acc.x * x + v.x * y;
            acc.y = acc.y * x + v.y * y;
            acc.z = acc.z * x + v.z * y;
            acc.w = acc.w * x + v.w * y;
        }
    };
    auto load = [&](int k, int r, float2& ml, float4& v) {
        const float* const p = part_of(k);
        ml = *reinterpret_cast<const float2*>(p + kPairRows * D + 2 * r);
        v = *reinterpret_cast<const float4*>(p + (d4 * kPairRows + r) * 4);
    };
    auto store = [&](int r, const Sum& s) {
        const float inv = 1.f / s.sum;
        const int row = join.first_row + r, token = row / a.group, hq = join.head * a.group + row - token * a.group;
        __half* const dst = a.out + (join.token + token) * a.out_stride + static_cast<long>(hq) * D + 4 * d4;
        const uint2 four = make_uint2(pack_half2(s.acc.x * inv, s.acc.y * inv), pack_half2(s.acc.z * inv, s.acc.w * inv));
        if (reinterpret_cast<uintptr_t>(dst) % 8 == 0) *reinterpret_cast<uint2*>(dst) = four;
        else {
            dst[0] = __ushort_as_half(static_cast<unsigned short>(four.x));
            dst[1] = __ushort_as_half(static_cast<unsigned short>(four.x >> 16));
            dst[2] = __ushort_as_half(static_cast<unsigned short>(four.y));
            dst[3] = __ushort_as_half(static_cast<unsigned short>(four.y >> 16));
        }
        if (a.lse && d4 == 0) a.lse[(join.token + token) * static_cast<long>(a.heads * a.group) + hq] = (s.top - kOffset + log2f(s.sum)) * 0.6931471805599453f;
    };
    const Sum none{-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
    if (ROWS > 1 && parts == 2) {
        float2 ml[ROWS][2];
        float4 v[ROWS][2];
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k) load(k, min(r0 + kJoinRows * i, join.rows - 1), ml[i][k], v[i][k]);
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            if (r0 + kJoinRows * i >= join.rows) break;
            Sum s = none;
            s.add(ml[i][0], v[i][0]);
            s.add(ml[i][1], v[i][1]);
            store(r0 + kJoinRows * i, s);
        }
        return;
    }
#pragma unroll 1
    for (int r = r0; r < min(join.rows, r0 + kJoinRows * ROWS); r += kJoinRows) {
        Sum s = none;
        for (int base = 0; base < parts; base += 8) {
            float2 ml[8];
            float4 v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) load(min(base + k, parts - 1), r, ml[k], v[k]);
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (base + k < parts) s.add(ml[k], v[k]);
        }
        store(r, s);
    }
}

template <int D, bool TREE>
void launch_typed(PagedAttnArgs a, long max_rows, void* scratch, int sms, cudaStream_t st) {
    a.joins = static_cast<PagedJoin*>(scratch);
    a.partial = reinterpret_cast<float*>(static_cast<char*>(scratch) + (sms * sizeof(PagedJoin) + 255) / 256 * 256);
    static std::atomic<unsigned long long> set{0};
    allow_shared_memory(paged_prompt_kernel<D, TREE>, Shape<D>::kSmem, set);
    launch_pdl_carved(paged_prompt_kernel<D, TREE>, dim3(static_cast<unsigned int>(sms)), dim3(kThreads), Shape<D>::kSmem, 100, st, a);
    const auto join = [&](auto kernel, int rows) {
        launch_pdl_carved(kernel, dim3(static_cast<unsigned int>(sms), static_cast<unsigned int>((std::min<long>(kPairRows, max_rows) + rows - 1) / rows)), dim3(kJoinRows * D / 4), 0, 100, st, a);
    };
    if (max_rows >= kPairRows) join(paged_prompt_join_kernel<D, 4>, 4 * kJoinRows);
    else join(paged_prompt_join_kernel<D, 1>, kJoinRows);
}

}  // namespace

size_t paged_prompt_scratch_bytes(int dim, int sms) {
    return (sms * sizeof(PagedJoin) + 255) / 256 * 256 + static_cast<size_t>(sms) * 2 * kPairRows * (static_cast<size_t>(dim) + 2) * sizeof(float);
}
void launch_paged_prompt(PagedAttnArgs a, int dim, long max_rows, void* scratch, int sms, cudaStream_t st) {
    if (dim == 64) launch_typed<64, false>(a, max_rows, scratch, sms, st);
    else launch_typed<128, false>(a, max_rows, scratch, sms, st);
}
void launch_paged_tree_attention(PagedAttnArgs a, int dim, long max_rows, void* scratch, int sms, cudaStream_t st) {
    a.few_rows = 0;
    if (dim == 64) launch_typed<64, true>(a, max_rows, scratch, sms, st);
    else launch_typed<128, true>(a, max_rows, scratch, sms, st);
}

}  // namespace tq
