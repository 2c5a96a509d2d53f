// The paged 8-bit KV cache: how it lies in memory, and what its kernels share.
//
// A page holds P tokens of every KV head.  The piece of a page that belongs to one head is one block of memory:
//
//   [keys P x D bytes][values P x D bytes][key scale, value scale, 24 bytes unused]
//
// so that a copy engine fetches a head's tokens of a page in three contiguous pieces and neither the number of heads nor the
// order of the pages matters.  A byte is code + 128, code -127 .. 127; the value is code * scale, the scale a power of two
// (or NaN: the block received a value that was not finite).  Powers of two make every product with a scale exact, a code that
// is rounded again when its block's scale grows loses half a step at most, and scales of different pages are taken together
// inside a matrix product without a rounding.
//
// The 16-byte chunks of a token's row stand in an order that depends on the token (key_chunk, value_chunk): the attention
// kernel's warps read the rows of eight tokens at once from shared memory, which lie a multiple of 64 bytes apart, and would meet
// in the same banks otherwise.
#pragma once

#include <atomic>
#include <cstdint>

#include "tq_common.cuh"

namespace tq {

constexpr int kPagedMaxRequests = 4096;
constexpr int kPagedMinExponent = -100;
constexpr int kPagedTail = 32;   // bytes behind a block's codes

__host__ __device__ __forceinline__ size_t paged_block_bytes(int page_tokens, int dim) {
    return 2 * static_cast<size_t>(page_tokens) * dim + kPagedTail;
}
// Where chunk c (16 dims) of a token's keys or values stands in its row.
template <int D>
__device__ __forceinline__ int key_chunk(int token, int c) {
    if constexpr (D == 128) return c ^ ((token & 1) << 2);
    else return c;
}
template <int D>
__device__ __forceinline__ int value_chunk(int token, int c) {
    if constexpr (D == 128) return c ^ (((token >> 1) & 3) << 1);
    else return c ^ ((token >> 1) & 3);
}

// What the host says of a plan: its requests, its tokens and one request's at most.
struct PagedSizes {
    int n, tokens, most;
};
// What the device keeps of the last plan, beside the arrays of PagedBatch.
struct __align__(16) PagedHeader {
    int free_pages;      // pages on the stack
    int requests, tokens, pieces;   // of the plan (all 0 where it was refused)
    PagedSizes sizes;    // n below 0: a truncation came behind it
    int unused;
};
// A run of new tokens in one page.
struct PagedPiece {
    int token, count, page, offset;
};
// Device arrays of a cache that its kernels read (and the plan writes).
struct PagedBatch {
    PagedHeader* header;
    int* lengths;          // [max_requests] tokens that each row of the tables holds
    int* tables;           // [max_requests][max_pages]
    int* stack;            // [num_pages] free pages, the next ones last
    int* rows;             // [max_requests] of the plan: row of the tables, first token, tokens held with the new ones
    int* starts;           // (+ 1)
    int* held;
    PagedPiece* pieces;
    int max_requests, max_pages, num_pages, page_tokens, max_pieces;
};

// Status codes of the paged cache's kernels.
enum PagedStatus : unsigned int {
    kPagedOk = 0,
    kPagedBadRow = 1,      // a row outside the tables, or twice
    kPagedBadCount = 2,    // a negative count, one above max_count, or more tokens in all than announced
    kPagedLongRequest = 3, // a request would need more pages than a table's row holds
    kPagedNoPages = 4,     // not enough free pages
    kPagedBadLength = 5,   // truncation to a length that the request does not have
    kPagedBadPage = 6,     // a page number outside the cache
    kPagedWait = 7,        // a bounded wait ran out
    kPagedOtherPlan = 8    // the plan on the device is not the one that a launch was made for
};

// Lets a kernel have so much dynamic shared memory, once for each device (`set`: those that have been).
template <typename Kernel>
void allow_shared_memory(Kernel kernel, size_t bytes, std::atomic<unsigned long long>& set) {
    int device = 0;
    TQ_CUDA(cudaGetDevice(&device));
    const unsigned long long bit = 1ull << (device & 63);
    if (device < 64 && (set.load(std::memory_order_relaxed) & bit)) return;
    TQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)));
    set.fetch_or(bit, std::memory_order_relaxed);
}

// ---- launches (tq_paged_plan.cu) ---------------------------------------------------------------
struct PagedPlanArgs {
    PagedBatch b;
    const int* rows;      // or null: 0, 1, ...
    const int* counts;
    int n, tokens, max_count;
    int* starts;          // outputs, any of them null
    int* lengths;
    int* slots;
    int* positions;
    int* tables;
    int tables_width;
    unsigned int* status;
    int sms;
};
void launch_paged_plan(const PagedPlanArgs& a, cudaStream_t st);
// counts: the lengths to keep
void launch_paged_truncate(const PagedPlanArgs& a, cudaStream_t st);
void launch_paged_init(uint8_t* layer, size_t blocks, size_t block_bytes, cudaStream_t st);

struct PagedAppendArgs {
    const PagedHeader* header;
    const PagedPiece* pieces;
    uint8_t* layer;
    const void* keys;
    const void* values;
    long key_stride, value_stride;   // elements from token to token
    int heads, page_tokens;
    PagedSizes sizes;
    unsigned int* status;
};
void launch_paged_append(const PagedAppendArgs& a, int dim, bool half, cudaStream_t st);

struct PagedReadArgs {
    const uint8_t* layer;
    const int* pages;
    void* keys;
    void* values;
    int n, heads, page_tokens, num_pages;
    unsigned int* status;
};
void launch_paged_read(const PagedReadArgs& a, int dim, bool half, cudaStream_t st);

// ---- attention (tq_paged_attention.cu) -----------------------------------------------------------
// An item that several CTAs share, as the CTA in which it begins leaves it for the kernel that adds the parts up.
struct PagedJoin {
    int last;        // the CTA in which it ends; 0: nothing to join (CTA 0 is never a last one)
    int cta;         // the one in which it begins
    int token;       // first token of its request
    int first_row;   // rows (token-major: row = token * group + head of the group) first_row ..
    int rows;        // ... and how many
    int head;        // KV head
};
struct PagedAttnArgs {
    PagedBatch b;
    const uint8_t* layer;
    const __half* q;
    __half* out;
    float* lse;          // or null
    long q_stride, out_stride;
    PagedSizes sizes;
    int heads, group, window, page_shift;
    int few_rows;        // requests of more query rows (new tokens times the group) go through tq_paged_prompt.cu
    float scale_log2;    // softmax scale times log2(e)
    float* partial;
    PagedJoin* joins;
    int join_items;      // few rows: entries of `joins` where each item has one (0: one for each CTA)
    unsigned int* status;
};
size_t paged_attn_scratch_bytes(int dim, int sms);
// The requests of at most a.few_rows rows, which are kFewRows or, where no request has more (max_rows), fewer.
constexpr int kFewRows = 16;
void launch_paged_attention(PagedAttnArgs a, int dim, int max_rows, void* scratch, int sms, cudaStream_t st);
// The others (tq_paged_prompt.cu).
size_t paged_prompt_scratch_bytes(int dim, int sms);
void launch_paged_prompt(PagedAttnArgs a, int dim, long max_rows, void* scratch, int sms, cudaStream_t st);

// ---- what the attention kernels share -------------------------------------------------------------
namespace paged_device {

// Requests and pieces of the plan on the device; none, with a status, where it is of other sizes than the launch (a captured step came between a plan
// and the call): the launch's grid, its choice of kernels and the caller's rows need not fit it.
struct Planned {
    int requests, pieces;
};
__device__ __forceinline__ Planned planned(const PagedHeader* header, const PagedSizes& sizes, unsigned int* status) {
    const int4 plan = reinterpret_cast<const int4*>(header)[0], made = reinterpret_cast<const int4*>(header)[1];   // (both on their way at once)
    if (made.x == sizes.n && made.y == sizes.tokens && made.z == sizes.most) return {plan.y, plan.w};
    if (blockIdx.x == 0 && threadIdx.x == 0) raise_status(status, kPagedOtherPlan);
    return {0, 0};
}

constexpr uint32_t kPagedWaitLimit = 400u * 1000 * 1000;   // cycles: 0.2 s at 2 GHz

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Bounded wait; gives up when another thread has.  (Few instructions: there is one behind every step of the kernels.  The limit is in clock cycles: reading
// the global timer takes longer than most waits, and a waiting warp does not see its barrier meanwhile.)
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile unsigned int* abort_flag) {
    uint32_t begin = 0;
    for (uint32_t spin = 0;; ++spin) {
        uint32_t done;
        asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                     : "=r"(done) : "r"(bar), "r"(parity) : "memory");
        if (done) return true;
        if ((spin & 255) == 255) {
            uint32_t now;
            asm volatile("mov.u32 %0, %%clock;" : "=r"(now));
            if (spin == 255) begin = now;
            if (*abort_flag || now - begin > kPagedWaitLimit) return false;
        }
    }
}
// Eight halves at any even address, out of the way of the code that runs all the time.
__device__ __noinline__ inline void store_halves_anywhere(__half* p, uint4 v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        p[2 * k] = __ushort_as_half(static_cast<unsigned short>(w[k]));
        p[2 * k + 1] = __ushort_as_half(static_cast<unsigned short>(w[k] >> 16));
    }
}
__device__ __noinline__ inline uint4 load_halves_anywhere(const __half* p) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = __half_as_ushort(p[2 * k]) | static_cast<uint32_t>(__half_as_ushort(p[2 * k + 1])) << 16;
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

}  // namespace paged_device

}  // namespace tq
