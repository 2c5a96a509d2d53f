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
// tokens' values 2^-15 of the largest one at the very worst, 1/16 of the result's rounding.
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

// instruction descriptor: D fp32, A and B fp16, both K-major, M = 128, N = n
__host__ __device__ constexpr uint32_t instr_desc(uint32_t n) { return (1u << 4) | ((n >> 3) << 17) | (static_cast<uint32_t>(kRows >> 4) << 24); }
// shared-memory descriptor: K-major, no swizzle, 128 bytes from core matrix to core matrix along K, `group` from 8 rows to the next 8
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t group) {
    return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(128u >> 4) << 16) | (static_cast<uint64_t>(group >> 4) << 32) | (1ull << 46);
}
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0;\n  tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p; }"
                 : : "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u) : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0;\n  tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p; }"
                 : : "r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u) : "memory");
}
__device__ __forceinline__ void umma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(p));
    return p != 0;
}
template <int N>
__device__ __forceinline__ void take_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void give_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void publish_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
          "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]),
          "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr));
}
// Waits for this thread's loads; the registers of one of them go through it, so that nothing that uses them comes earlier.
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]),
                   "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]),
                   "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        : : "r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
            "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        : : "r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
            "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]),
            "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A request of many rows; all lanes of a warp hold the same.
struct Request {
    int row, start, count, held, rows;
    __device__ __forceinline__ int first() const { return held - count; }
    __device__ __forceinline__ int pairs() const { return (rows + kPairRows - 1) / kPairRows; }
    // tiles of the cache that the rows of a pair see
    __device__ __forceinline__ void tiles(const PagedAttnArgs& a, int pair, int& lo, int& hi) const {
        const int last = first() + (min(rows, (pair + 1) * kPairRows) - 1) / a.group;
        hi = last / kTokens + 1;
        lo = a.window > 0 ? max(0, first() + pair * kPairRows / a.group - a.window + 1) / kTokens : 0;
    }
};
// The first request of many rows from i on (lanes look at 32 at a time); n if there is none.
__device__ __forceinline__ int next_request(const PagedAttnArgs& a, int i, int n, int lane, Request& r) {
    for (int base = i; base < n; base += 32) {
        const int mine = min(base + lane, n - 1);
        Request x;
        x.row = a.b.rows[mine];
        x.start = a.b.starts[mine];
        x.count = a.b.starts[mine + 1] - x.start;
        x.held = a.b.held[mine];
        const bool many = base + lane < n && x.count * a.group > a.few_rows;
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
__device__ __forceinline__ long long request_tiles(const PagedAttnArgs& a, const Request& r, int lane) {
    long long sum = 0;
    for (int p = lane; p < r.pairs(); p += 32) {
        int lo, hi;
        r.tiles(a, p, lo, hi);
        sum += hi - lo + kItemUnits;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
}

// A CTA's share of the units: (request, KV head, pair, tile), the tile running fastest.
struct Walker {
    Request r;
    int i, n, head, pair, lo, hi, tile;
    int before;          // units of kItemUnits that come in front of the present tile
    long long left;
    __device__ __forceinline__ void place(const PagedAttnArgs& a, int request, int requests, long long skip, long long units, int lane) {
        n = requests;
        left = units;
        i = next_request(a, request, n, lane, r);
        long long sum;
        while (i < n && skip >= (sum = request_tiles(a, r, lane)) * a.heads) {
            skip -= sum * a.heads;
            i = next_request(a, i + 1, n, lane, r);
        }
        if (i >= n) {   // (not with a share of units that exist)
            left = 0;
            return;
        }
        head = static_cast<int>(skip / sum);
        skip -= head * sum;
        for (int base = 0;; base += 32) {   // the pair in which the rest lies
            int l = 0, h = 0;
            if (base + lane < r.pairs()) r.tiles(a, base + lane, l, h);
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
                i = next_request(a, i + 1, n, lane, r);
                if (i >= n) return false;
            }
        }
        r.tiles(a, pair, lo, hi);
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
};
constexpr int kSegments = 4;
constexpr int kSegmentReaders = 30;   // warps: softmax, products, queries, keys, values

struct Bars {
    unsigned long long q_full[2], q_empty[2], s_full[2][2], p_full[2][2], o_done[2][2], o_empty[2], k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages], seg_full[kSegments], seg_empty[kSegments], done[2];
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

template <int D>
__global__ void __launch_bounds__(kThreads, 1) paged_prompt_kernel(const __grid_constant__ PagedAttnArgs a) {
    using S = Shape<D>;
    extern __shared__ __align__(1024) uint8_t s_mem[];
    __shared__ __align__(8) Bars s_bar;
    __shared__ long long s_sum[kWarps];
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
        for (int k = 0; k < kSegments; ++k) {
            bar_init(bar(s_bar.seg_full[k]), 1);
            bar_init(bar(s_bar.seg_empty[k]), kSegmentReaders);
        }
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_wait_release();
    const int n = planned(a.b.header, a.sizes, a.status).requests;
    const int per = (n + kWarps - 1) / kWarps;
    {
        const int end = min(n, (warp + 1) * per);
        long long mine = 0;
        Request r;
        for (int i = next_request(a, warp * per, end, lane, r); i < end; i = next_request(a, i + 1, end, lane, r)) mine += request_tiles(a, r, lane) * a.heads;
        if (lane == 0) s_sum[warp] = mine;
    }
    __syncthreads();
    long long total = 0;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) total += s_sum[k];
    const long long ctas = min(static_cast<long long>(gridDim.x), total), c = blockIdx.x;
    if (tid == 0) a.joins[c].last = 0;
    if (c >= ctas) return;
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)), "r"(kTmemAll) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        fence_before();
    }
    __syncthreads();
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
        while (next_segment()) {
            const Segment& at = s_seg[seg_n % kSegments];
            const int tiles = at.tiles, tile0 = at.tile;
            if (t == 0 || at.two()) {
                const int row = at.row0 + t * kRows + r_in, in_row = min(row, at.rows - 1);
                const int token = at.start + in_row / a.group, hq = at.head * a.group + in_row % a.group, pos = at.first + in_row / a.group;
                const bool live = row < at.rows;
                const int oldest = a.window > 0 ? max(0, pos - a.window + 1) : 0;
                // A warp without rows: it keeps the others' count (16 requests of 35 rows: 48 us, 56 with the softmax of what is not there)
                const bool idle = at.row0 + t * kRows + 32 * (warp & 3) >= at.rows;
                // O is in units of vref: the largest of the values' scales that the row has seen (vseen), or the tile's where it sees only part of
                // the tile and the rest is larger.  It comes down again behind such a tile: a window that begins there has all its other tokens in
                // front.
                float m = -INFINITY, l = 0.f, vref = 0.f, vseen = 0.f;
                for (int j = 0; j < tiles; ++j) {
                    const uint32_t ref = (count + j) & (kRefs - 1), n = done + j;
                    if (!wait(s_bar.s_full[t][n & 1], (n >> 1) & 1)) break;
                    if (idle) {
                        if (lane == 0) bar_arrive(bar(s_bar.p_full[t][n & 1]));
                        continue;
                    }
                    fence_after();
                    const uint32_t t_s = t_s0 + (n & 1) * kTokens;
                    uint32_t x[32], y[32];
                    const float kref = s_kref[ref], vref_here = s_vref[ref];
                    tmem_ld(t_s, x);
                    tmem_ld(t_s + 32, y);
                    const int tb = (tile0 + j) * kTokens;
                    const float f = fmaxf(kref * a.scale_log2, 1.1754944e-38f);   // (not 0: minus infinity times it)
                    const int newest = pos - tb, eldest = oldest - tb;   // columns eldest .. newest are seen
                    float vt = newest >= 0 && eldest < kTokens ? vref_here : 0.f, vpart = vt;   // (what a row does not see leaves its unit alone)
                    tmem_ld_wait(x);
                    tmem_ld_wait(y);
                    if (__any_sync(0xffffffffu, newest < kTokens - 1 || eldest > 0)) {
                        // a bit for each column
                        const uint64_t seen = (newest >= 63 ? ~0ull : newest < 0 ? 0ull : (2ull << newest) - 1) & (eldest <= 0 ? ~0ull : eldest > 63 ? 0ull : ~0ull << eldest);
                        const uint32_t lo = static_cast<uint32_t>(seen), hi = static_cast<uint32_t>(seen >> 32);
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
                    weights(x, t_s);
                    weights(y, t_s + 16);
                    const float2 both_sums = unpack2(add2(sums[0], sums[1]));
                    const float sum = both_sums.x + both_sums.y;
                    l = fmaf(sum, exp2_approx(-lower), l);
                    if (moves && j > 0) {   // O to the new reference: behind the weights, which take as long as the products that it waits for
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
                done += tiles;
                if (wait(s_bar.o_done[t][(done - 1) & 1], ((done - 1) >> 1) & 1)) {
                    fence_after();
                    const bool begins = at.begins, ends = at.ends;
                    const float unit = vref * (1.f / kHeadroom);
                    uint32_t x[32];
                    if (begins && ends) {
                        const float inv = unit / l;
                        __half* const dst = a.out + token * a.out_stride + static_cast<long>(hq) * D;
#pragma unroll 1
                        for (int q = 0; q < D / 32; ++q) {
                            tmem_ld(t_o + 32 * q, x);
                            tmem_ld_wait(x);
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
                        for (int q = 0; q < D / 32; ++q) {
                            tmem_ld(t_o + 32 * q, x);
                            tmem_ld_wait(x);
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
                    if (lane == 0) bar_arrive(bar(s_bar.o_empty[t]));
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
#pragma unroll 1
                for (int j = 0; j < tiles; ++j, ++turns) {
                    const uint32_t stage = turns % kStages, turn = (turns / kStages) & 1;
                    if (!until(first ? s_bar.k_full[stage] : s_bar.v_full[stage], turn)) break;
#pragma unroll 1
                    for (int t = 0; t < pair; ++t) {
                        const uint32_t nt = t ? n1 : n0, place = nt & 1, t_s = tmem + (2 * t + place) * kTokens;
                        if (first) {
                            if (j == 0 && !until(s_bar.q_full[t], (items >> t) & 1)) break;
                            // P of two tiles before was where these scores go
                            if (nt >= 2 && !until(s_bar.o_done[t][place], ((nt >> 1) - 1) & 1)) break;
                            fence_after();
                            const uint64_t q = q_desc + t * (S::kQBytes >> 4), k = k_desc + stage * (S::kKBytes >> 4);
#pragma unroll
                            for (int s = 0; s < D / 16; ++s) umma_ss(t_s, q + 16 * s, k + 16 * s, kIdescS, s > 0);
                            umma_commit(bar(s_bar.s_full[t][place]));
                            if (j + 1 == tiles) umma_commit(bar(s_bar.q_empty[t]));
                        } else {
                            if (j == 0 && !until(s_bar.o_empty[t], ((items >> t) & 1) ^ 1)) break;
                            if (!until(s_bar.p_full[t][place], (nt >> 1) & 1)) break;
                            fence_after();
                            const uint64_t v = v_desc + stage * (S::kVBytes >> 4);
#pragma unroll
                            for (int s = 0; s < kTokens / 16; ++s) umma_ts(tmem + 4 * kTokens + t * D, t_s + 8 * s, v + 16 * s, kIdescO, j > 0 || s > 0);
                            umma_commit(bar(s_bar.o_done[t][place]));
                        }
                        if (t) ++n1; else ++n0;
                    }
                    if (!go) break;
                    umma_commit(bar(first ? s_bar.k_empty[stage] : s_bar.v_empty[stage]));
                }
                items ^= pair == 2 ? 3u : 1u;
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
            const long long u0 = total * c / ctas, u1 = total * (c + 1) / ctas;
            Walker at;
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
                    const long long last_unit = u1 - at.left + at.before + (at.hi - at.tile) - 1;
                    s_seg[seg_n % kSegments] = {at.r.row, at.r.start, at.r.first(), at.r.held, at.r.rows, at.pair * kPairRows, at.head, at.tile, tiles, at.tile == at.lo,
                                                at.tile + tiles == at.hi, static_cast<int>(((last_unit + 1) * ctas - 1) / total)};
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
            if (keys) {
                // lane = (row of 8, chunk of 4)
                const uint32_t ref = largest_scale(key_bits);
                const __half2 fa = __float2half2_rn(code_factor(__shfl_sync(0xffffffffu, key_bits, page), ref)), off = __hmul2(fa, __float2half2_rn(-1152.f));
                uint8_t* const dst = s_mem + S::kK + stage * S::kKBytes + 2 * w * S::kRowGroup + (lane & 7) * 16;
#pragma unroll 1
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
                        s_vref[now.n & (kRefs - 1)] = __uint_as_float(value_ref);
                    }
                }
            } else {
                // a lane takes four dims of eight tokens
                constexpr int kLanes = D / 4, kGroups = 32 / kLanes;   // groups of 8 tokens side by side in a warp
                const int d4 = lane % kLanes;
                const __half2 fa = __float2half2_rn(code_factor(__shfl_sync(0xffffffffu, value_bits, page), value_ref)), off = __hmul2(fa, __float2half2_rn(-1152.f));
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
            step(now);
            if (now.tiles > 0) step(now);
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

template <int D>
void launch_typed(PagedAttnArgs a, long max_rows, void* scratch, int sms, cudaStream_t st) {
    a.joins = static_cast<PagedJoin*>(scratch);
    a.partial = reinterpret_cast<float*>(static_cast<char*>(scratch) + (sms * sizeof(PagedJoin) + 255) / 256 * 256);
    static std::atomic<unsigned long long> set{0};
    allow_shared_memory(paged_prompt_kernel<D>, Shape<D>::kSmem, set);
    launch_pdl_carved(paged_prompt_kernel<D>, dim3(static_cast<unsigned int>(sms)), dim3(kThreads), Shape<D>::kSmem, 100, st, a);
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
    if (dim == 64) launch_typed<64>(a, max_rows, scratch, sms, st);
    else launch_typed<128>(a, max_rows, scratch, sms, st);
}

}  // namespace tq
