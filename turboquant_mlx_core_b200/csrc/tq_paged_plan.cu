// The paged 8-bit KV cache's bookkeeping (block tables, slot maps and positions from the requests' token counts), the quantising
// write of new keys and values, and the read-back of pages.  The reference keeps one growing store per sequence whose length
// the host knows (include/turboquant/kv_cache.h:42-133); here many requests share pages and the lengths live on the device, so
// that a decode loop with drafts never waits for the host.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>

#include "tq_common.cuh"
#include "tq_host.hpp"
#include "tq_paged.cuh"

namespace tq {

namespace {

namespace cg = cooperative_groups;

constexpr int kPlanThreads = 1024;
constexpr int kPlanPerThread = kPagedMaxRequests / kPlanThreads;

// Exclusive sums over the CTA of three numbers per thread; the totals come back in `all`.
__device__ __forceinline__ void block_sums(long long (&v)[3], long long (&all)[3]) {
    __shared__ long long s_warp[32][3];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long mine[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        mine[k] = v[k];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long t = __shfl_up_sync(0xffffffffu, v[k], o);
            if (lane >= o) v[k] += t;
        }
        if (lane == 31) s_warp[warp][k] = v[k];
    }
    __syncthreads();
    if (warp == 0) {
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            long long t = s_warp[lane][k];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long u = __shfl_up_sync(0xffffffffu, t, o);
                if (lane >= o) t += u;
            }
            s_warp[lane][k] = t;
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        v[k] += (warp ? s_warp[warp - 1][k] : 0) - mine[k];
        all[k] = s_warp[31][k];
    }
}

// The last i of 0 .. n - 1 with base[i] <= x (base ascending, base[0] = 0): of several equal ones the last, which is the one with something in it.
__device__ __forceinline__ int owner_of(const int* base, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (base[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Rows that were named twice: a bit each.
__device__ __forceinline__ void clear_seen(unsigned int* seen) {
    for (int i = threadIdx.x; i < kPagedMaxRequests / 32; i += kPlanThreads) seen[i] = 0;
}
__device__ __forceinline__ bool seen_before(unsigned int* seen, int row) {
    const unsigned int bit = 1u << (row & 31);
    return (atomicOr(&seen[row >> 5], bit) & bit) != 0;
}

// Every CTA reads all requests and takes the sums over them (4096 at most, from the L2 cache), and the CTAs share the output: tokens, pieces, new
// pages and the tables' copy, each element found by a binary search in the sums.  All or nothing: a batch that does not fit leaves the cache as it
// was, an empty plan and a status.  COMMIT: one cluster, behind whose barrier nobody reads the lengths and the number of free pages any more, which
// then change.  It is bound by latency: a launch, two dependent loads, the sums' barriers.  Much output is written by as many CTAs as there are SMs
// (OUTPUT), with no barrier between them, in front of a cluster that only commits (61 prompts of up to 8192 tokens, 3 MB: 54 us with one cluster of
// eight for both, 13 so).
template <bool OUTPUT, bool COMMIT>
__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(PagedPlanArgs a) {
    pdl_wait_release();
    behind_wait(a.rows, a.counts);
    extern __shared__ int s_plan[];
    __shared__ unsigned int s_seen[kPagedMaxRequests / 32];
    __shared__ unsigned int s_error;
    // (the grid is the cluster where it commits)
    const int rank = static_cast<int>(blockIdx.x), ctas = static_cast<int>(gridDim.x);
    const int n = a.n, P = a.b.page_tokens, tid = threadIdx.x;
    int* const s_row = s_plan;             // [n]
    int* const s_old = s_row + n;          // [n]
    int* const s_start = s_old + n;        // [n + 1]
    int* const s_page = s_start + n + 1;   // [n + 1] new pages in front of the request's
    int* const s_piece = s_page + n + 1;   // [n + 1]
    clear_seen(s_seen);
    if (tid == 0) s_error = kPagedOk;
    __syncthreads();
    const int free_before = *static_cast<volatile int*>(&a.b.header->free_pages);

    const int per = (n + kPlanThreads - 1) / kPlanThreads, i0 = tid * per;
    int row[kPlanPerThread], old[kPlanPerThread], count[kPlanPerThread];
    long long sums[3] = {0, 0, 0}, all[3];
#pragma unroll
    for (int k = 0; k < kPlanPerThread; ++k) {
        row[k] = old[k] = count[k] = 0;
        if (k >= per || i0 + k >= n) continue;
        row[k] = a.rows ? a.rows[i0 + k] : i0 + k;
        count[k] = a.counts[i0 + k];
        unsigned int bad = kPagedOk;
        if (row[k] < 0 || row[k] >= a.b.max_requests || seen_before(s_seen, row[k])) bad = kPagedBadRow;
        else if (count[k] < 0 || count[k] > a.max_count) bad = kPagedBadCount;
        else {
            old[k] = a.b.lengths[row[k]];
            if (static_cast<long long>(old[k]) + count[k] > static_cast<long long>(a.b.max_pages) * P) bad = kPagedLongRequest;
        }
        if (bad != kPagedOk) {
            atomicMax(&s_error, bad);
            row[k] = old[k] = count[k] = 0;   // (nothing below goes by what it names)
            continue;
        }
        const int now = old[k] + count[k];
        sums[0] += count[k];
        sums[1] += (now + P - 1) / P - (old[k] + P - 1) / P;
        if (count[k]) sums[2] += (now - 1) / P - old[k] / P + 1;
    }
    block_sums(sums, all);   // (its barriers publish s_error)
    unsigned int error = s_error;
    if (error == kPagedOk && all[0] > a.tokens) error = kPagedBadCount;
    if (error == kPagedOk && all[1] > free_before) error = kPagedNoPages;
    const bool ok = error == kPagedOk;
    const int tokens = ok ? static_cast<int>(all[0]) : 0, pages = ok ? static_cast<int>(all[1]) : 0, pieces = ok ? static_cast<int>(all[2]) : 0;
    int at = static_cast<int>(sums[0]), page = static_cast<int>(sums[1]), piece = static_cast<int>(sums[2]);
#pragma unroll
    for (int k = 0; k < kPlanPerThread; ++k) {
        const int i = i0 + k;
        if (k >= per || i >= n) continue;
        if (!ok) count[k] = at = page = piece = 0;
        s_row[i] = row[k];
        s_old[i] = old[k];
        s_start[i] = at;
        s_page[i] = page;
        s_piece[i] = piece;
        const int now = old[k] + count[k];
        at += count[k];
        page += (now + P - 1) / P - (old[k] + P - 1) / P;
        if (count[k]) piece += (now - 1) / P - old[k] / P + 1;
    }
    if (tid == 0) {
        s_start[n] = tokens;
        s_page[n] = pages;
        s_piece[n] = pieces;
    }
    if constexpr (COMMIT) cg::this_cluster().sync();   // every CTA has read the lengths and the number of free pages (and its own sums are complete)
    else __syncthreads();

    // page `idx` of request i, before the plan's writes to the tables
    auto page_of = [&](int i, int idx) {
        const int had = (s_old[i] + P - 1) / P;
        return idx < had ? a.b.tables[static_cast<size_t>(s_row[i]) * a.b.max_pages + idx] : a.b.stack[free_before - 1 - (s_page[i] + idx - had)];
    };
    const int t0 = rank * kPlanThreads + tid, step = ctas * kPlanThreads;
    if constexpr (COMMIT) {
        for (int t = t0; t < n; t += step) {
            const int now = s_old[t] + s_start[t + 1] - s_start[t];
            a.b.rows[t] = s_row[t];
            a.b.starts[t] = s_start[t];
            a.b.held[t] = now;
            if (ok) a.b.lengths[s_row[t]] = now;
            if (a.starts) a.starts[t] = s_start[t];
            if (a.lengths) a.lengths[t] = now;
        }
        if (t0 == 0) {
            a.b.starts[n] = tokens;
            if (a.starts) a.starts[n] = tokens;
            *a.b.header = {free_before - pages, ok ? n : 0, tokens, pieces, {n, a.tokens, min(a.max_count, a.tokens)}, 0};
            if (!ok) raise_status(a.status, error);
        }
    }
    if constexpr (OUTPUT) {
        for (int t = t0; t < pages; t += step) {
            const int i = owner_of(s_page, n, t), idx = (s_old[i] + P - 1) / P + t - s_page[i];
            a.b.tables[static_cast<size_t>(s_row[i]) * a.b.max_pages + idx] = a.b.stack[free_before - 1 - t];
        }
        for (int t = t0; t < pieces; t += step) {
            const int i = owner_of(s_piece, n, t), idx = s_old[i] / P + t - s_piece[i], count_i = s_start[i + 1] - s_start[i];
            const int first = max(s_old[i], idx * P), last = min(s_old[i] + count_i, (idx + 1) * P);
            a.b.pieces[t] = {s_start[i] + first - s_old[i], last - first, page_of(i, idx), first - idx * P};
        }
        if (a.slots || a.positions) {
            for (int t = t0; t < a.tokens; t += step) {
                int slot = -1, position = 0;
                if (t < tokens) {
                    const int i = owner_of(s_start, n, t);
                    position = s_old[i] + t - s_start[i];
                    const int idx = position / P;
                    if (a.slots) slot = page_of(i, idx) * P + position - idx * P;
                }
                if (a.slots) a.slots[t] = slot;
                if (a.positions) a.positions[t] = position;
            }
        }
        if (a.tables) {
            const long cells = static_cast<long>(n) * a.tables_width;
            for (long t = t0; t < cells; t += step) {
                const int i = static_cast<int>(t / a.tables_width), idx = static_cast<int>(t - static_cast<long>(i) * a.tables_width);
                const int has = (s_old[i] + s_start[i + 1] - s_start[i] + P - 1) / P;
                a.tables[t] = idx < has ? page_of(i, idx) : -1;
            }
        }
    }
}

// Requests give back what lies beyond a.counts[i] tokens; their pages go onto the stack so that a plan takes them off again in the same
// order.  The plan in force ends with it.
__global__ void __launch_bounds__(kPlanThreads) paged_truncate_kernel(PagedPlanArgs a) {
    pdl_wait_release();
    behind_wait(a.rows, a.counts);
    extern __shared__ int s_plan[];
    __shared__ unsigned int s_seen[kPagedMaxRequests / 32];
    __shared__ unsigned int s_error;
    const cg::cluster_group cluster = cg::this_cluster();
    const int rank = static_cast<int>(cluster.block_rank()), ctas = static_cast<int>(cluster.num_blocks());
    const int n = a.n, P = a.b.page_tokens, tid = threadIdx.x;
    int* const s_row = s_plan;            // [n]
    int* const s_keep = s_row + n;        // [n] pages that stay
    int* const s_page = s_keep + n;       // [n + 1] freed pages in front of the request's
    clear_seen(s_seen);
    if (tid == 0) s_error = kPagedOk;
    __syncthreads();
    const int free_before = *static_cast<volatile int*>(&a.b.header->free_pages);
    const int per = (n + kPlanThreads - 1) / kPlanThreads, i0 = tid * per;
    int row[kPlanPerThread], old[kPlanPerThread], keep[kPlanPerThread];
    long long sums[3] = {0, 0, 0}, all[3];
#pragma unroll
    for (int k = 0; k < kPlanPerThread; ++k) {
        row[k] = old[k] = keep[k] = 0;
        if (k >= per || i0 + k >= n) continue;
        row[k] = a.rows ? a.rows[i0 + k] : i0 + k;
        keep[k] = a.counts[i0 + k];
        unsigned int bad = kPagedOk;
        if (row[k] < 0 || row[k] >= a.b.max_requests || seen_before(s_seen, row[k])) bad = kPagedBadRow;
        else {
            old[k] = a.b.lengths[row[k]];
            if (keep[k] < 0 || keep[k] > old[k]) bad = kPagedBadLength;
        }
        if (bad != kPagedOk) {
            atomicMax(&s_error, bad);
            row[k] = old[k] = keep[k] = 0;
            continue;
        }
        sums[0] += (old[k] + P - 1) / P - (keep[k] + P - 1) / P;
    }
    block_sums(sums, all);
    const bool ok = s_error == kPagedOk;
    const int pages = ok ? static_cast<int>(all[0]) : 0;
    int page = static_cast<int>(sums[0]);
#pragma unroll
    for (int k = 0; k < kPlanPerThread; ++k) {
        const int i = i0 + k;
        if (k >= per || i >= n) continue;
        s_row[i] = row[k];
        s_keep[i] = (keep[k] + P - 1) / P;
        s_page[i] = ok ? page : 0;
        page += (old[k] + P - 1) / P - s_keep[i];
    }
    if (tid == 0) s_page[n] = pages;
    cluster.sync();
    const int t0 = rank * kPlanThreads + tid, step = ctas * kPlanThreads;
    if (ok) {
        for (int t = t0; t < n; t += step) a.b.lengths[s_row[t]] = a.counts[t];
        for (int t = t0; t < pages; t += step) {
            const int i = owner_of(s_page, n, t), idx = s_keep[i] + t - s_page[i];
            a.b.stack[free_before + pages - 1 - t] = a.b.tables[static_cast<size_t>(s_row[i]) * a.b.max_pages + idx];
        }
    }
    if (t0 == 0) {
        *a.b.header = {free_before + pages, 0, 0, 0, {-1, 0, 0}, 0};
        if (!ok) raise_status(a.status, s_error);
    }
}

// `ctas` CTAs, a cluster where there are 2 .. 8 of them and they are to be one.
template <typename Kernel>
void launch_cluster(Kernel kernel, int ctas, bool cluster, size_t smem, const PagedPlanArgs& a, cudaStream_t st, std::atomic<unsigned long long>& set) {
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned int>(ctas);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned int>(ctas));
    cfg.blockDim = dim3(kPlanThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = cluster && ctas > 1 ? 2 : 1;
    if (smem > 40 * 1024) allow_shared_memory(kernel, (5 * static_cast<size_t>(kPagedMaxRequests) + 3) * sizeof(int), set);
    TQ_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
}

// CTAs of a plan's cluster: one for every 4096 elements of output, up to 8 (the portable most); for more output than kOneCluster see the kernel.
constexpr long kOneCluster = 100000;
int plan_ctas(long elements) {
    int ctas = 1;
    while (ctas < 8 && static_cast<long>(ctas) * 4096 < elements) ctas *= 2;
    return ctas;
}

__global__ void __launch_bounds__(256) paged_init_kernel(uint8_t* layer, size_t blocks, size_t block_bytes) {
    const size_t codes = (block_bytes - kPagedTail) / 16;
    const uint4 none = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
    const float scale = __uint_as_float(static_cast<unsigned int>(127 + kPagedMinExponent) << 23);
    for (size_t b = blockIdx.x; b < blocks; b += gridDim.x) {
        uint4* const p = reinterpret_cast<uint4*>(layer + b * block_bytes);
        for (size_t i = threadIdx.x; i < codes; i += 256) p[i] = none;
        if (threadIdx.x == 0) {
            p[codes] = make_uint4(__float_as_uint(scale), __float_as_uint(scale), 0u, 0u);
            p[codes + 1] = make_uint4(0u, 0u, 0u, 0u);
        }
    }
}

// ---- the quantising write -------------------------------------------------------------------------

// Bits of the power of two with which a largest magnitude of these bits becomes a code of at most 127: 2^(x - 7) or 2^(x - 6) for a
// magnitude of [2^(x - 1), 2^x), the larger one where the smaller would give 127.5 or more.  NaN where it is not finite.
__device__ __forceinline__ unsigned int scale_bits(unsigned int top) {
    if (top >= 0x7f800000u) return 0x7fc00000u;
    const int x = static_cast<int>(top >> 23) - 126;
    const int e = max((top & 0x7fffffu) < 0x7f0000u ? x - 7 : x - 6, kPagedMinExponent);
    return static_cast<unsigned int>(e + 127) << 23;
}

// 16 values of a row as fp32; WIDE: rows are 16-byte aligned.
template <typename T, bool WIDE>
__device__ __forceinline__ void load16(float (&v)[16], const T* p) {
    if constexpr (!WIDE) {
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = static_cast<float>(p[j]);
    } else if constexpr (sizeof(T) == 2) {
        const uint4 a = reinterpret_cast<const uint4*>(p)[0], b = reinterpret_cast<const uint4*>(p)[1];
        float lo[8], hi[8];
        unpack_halves(a, lo);
        unpack_halves(b, hi);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] = lo[j];
            v[8 + j] = hi[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float4 f = reinterpret_cast<const float4*>(p)[j];
            v[4 * j] = f.x; v[4 * j + 1] = f.y; v[4 * j + 2] = f.z; v[4 * j + 3] = f.w;
        }
    }
}
// Codes of 16 values: round(v * inverse) + 128, to the nearest, ties to even (inverse is a power of two: the product is exact, but for what
// rounds to 0 anyway).
__device__ __forceinline__ uint4 encode16(const float (&v)[16], float inverse) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t b[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) b[k] = static_cast<uint32_t>(__float2int_rn(v[4 * j + k] * inverse) + 128);
        w[j] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void decode16(float (&v)[16], const uint4& c, float scale) {
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = static_cast<float>(static_cast<int>((w[j >> 2] >> (8 * (j & 3))) & 255u) - 128) * scale;
}

// A warp (for the few tokens of a decode step, four jobs to a CTA) or a CTA writes one piece's tokens of one head's keys or values: largest
// magnitude, scale, codes.  A thread takes 16 dims of ITER tokens, all asked for at once, which stay in registers (read twice, the second time from
// the caches, 67 thousand fp32 tokens of 8 heads took 145 us). Older tokens of the page are read only where its scale grows.
template <int D, typename T, bool WIDE, bool WARP, int ITER>
__global__ void __launch_bounds__(WARP ? 128 : 256) paged_append_kernel(PagedAppendArgs a) {
    constexpr int kThreads = WARP ? 32 : 256, kChunks = D / 16, kRows = kThreads / kChunks;
    pdl_wait_release();
    behind_wait(a.pieces, a.header, a.keys, a.values);
    const int lane = threadIdx.x & 31, tid = WARP ? lane : threadIdx.x;
    const long jobs = static_cast<long>(paged_device::planned(a.header, a.sizes, a.status).pieces) * a.heads * 2;
    const int P = a.page_tokens, c = tid % kChunks, r0 = tid / kChunks;
    const size_t block = paged_block_bytes(P, D);
    long job = blockIdx.x, stride = gridDim.x;
    if constexpr (WARP) {
        job = job * 4 + (threadIdx.x >> 5);
        stride *= 4;
    }
    __shared__ unsigned int s_top[8];
    for (; job < jobs; job += stride) {
        const bool second = (job & 1) != 0;
        const long rest = job >> 1;
        const int head = static_cast<int>(rest % a.heads);
        const PagedPiece piece = a.pieces[rest / a.heads];
        const long row_stride = second ? a.value_stride : a.key_stride;
        const T* const src = static_cast<const T*>(second ? a.values : a.keys) + piece.token * row_stride + static_cast<long>(head) * D + 16 * c;
        uint8_t* const dst = a.layer + (static_cast<size_t>(piece.page) * a.heads + head) * block;
        uint8_t* const codes = dst + (second ? static_cast<size_t>(P) * D : 0);
        float* const scale_at = reinterpret_cast<float*>(dst + 2 * static_cast<size_t>(P) * D) + (second ? 1 : 0);
        float v[ITER][16];
#pragma unroll
        for (int i = 0; i < ITER; ++i) load16<T, WIDE>(v[i], src + min(r0 + i * kRows, piece.count - 1) * row_stride);   // (rows behind the last: the last again)
        const unsigned int held = piece.offset ? __float_as_uint(*scale_at) : 0u;
        unsigned int top = 0;
#pragma unroll
        for (int i = 0; i < ITER; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) top = max(top, __float_as_uint(v[i][j]) & 0x7fffffffu);
        top = __reduce_max_sync(0xffffffffu, top);
        if constexpr (!WARP) {
            if (lane == 0) s_top[threadIdx.x >> 5] = top;
            __syncthreads();
#pragma unroll
            for (int k = 0; k < 8; ++k) top = max(top, s_top[k]);
        }
        const unsigned int scale = max(scale_bits(top), held);   // (as bits: NaN is above the finite ones, and stays)
        const bool finite = scale < 0x7f800000u;
        const float inverse = finite ? __uint_as_float((254u << 23) - scale) : 0.f;
        auto place = [&](int token) {
            return reinterpret_cast<uint4*>(codes + static_cast<size_t>(token) * D + 16 * (second ? value_chunk<D>(token, c) : key_chunk<D>(token, c)));
        };
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int r = r0 + i * kRows;
            if (r >= piece.count) continue;
            if (!finite) {
#pragma unroll
                for (int j = 0; j < 16; ++j) v[i][j] = 0.f;
            }
            *place(piece.offset + r) = encode16(v[i], inverse);
        }
        if (finite && piece.offset && scale != held) {
            const float ratio = __uint_as_float(held) * inverse;
            float old[16];
            for (int t = r0; t < piece.offset; t += kRows) {
                decode16(old, *place(t), 1.f);
                *place(t) = encode16(old, ratio);
            }
        }
        if (!WARP) __syncthreads();   // s_top, and the scale that was read, are everyone's until here
        else __syncwarp();
        if (tid == 0) *scale_at = __uint_as_float(scale);
    }
}

template <int D, typename T, bool WIDE>
void launch_append_typed(const PagedAppendArgs& a, cudaStream_t st) {
    // pieces that the plan can have: each of the requests begins and ends in a page of its own
    const long most = std::min<long>(a.sizes.tokens, a.sizes.tokens / a.page_tokens + 2L * a.sizes.n) * a.heads * 2;
    if (most == 0) return;
    constexpr int kWarpRows = 512 / D, kCtaRows = 4096 / D;   // tokens at a time
    const int longest = std::min(a.sizes.most, a.page_tokens);
    auto warps = [&](auto kernel) { launch_pdl(kernel, dim3(static_cast<unsigned int>(std::min<long>((most + 3) / 4, 1 << 20))), dim3(128), 0, st, a); };
    auto ctas = [&](auto kernel) { launch_pdl(kernel, dim3(static_cast<unsigned int>(std::min<long>(most, 1 << 20))), dim3(256), 0, st, a); };
    if (longest <= kWarpRows) warps(paged_append_kernel<D, T, WIDE, true, 1>);
    else if (longest <= 2 * kWarpRows) warps(paged_append_kernel<D, T, WIDE, true, 2>);
    else if (longest <= kCtaRows) ctas(paged_append_kernel<D, T, WIDE, false, 1>);
    else if (longest <= 2 * kCtaRows) ctas(paged_append_kernel<D, T, WIDE, false, 2>);
    else ctas(paged_append_kernel<D, T, WIDE, false, D == 128 ? 4 : 2>);
}

// ---- pages back -------------------------------------------------------------------------------------

// A CTA per page and head: its codes come in rows of 16-byte chunks and go out in the tensor's order [page][token][head][dim].
template <int D, typename T>
__global__ void __launch_bounds__(256) paged_read_kernel(PagedReadArgs a) {
    pdl_wait_release();
    behind_wait(a.pages, a.layer);
    constexpr int kChunks = D / 16;
    const int P = a.page_tokens, i = blockIdx.x / a.heads, head = blockIdx.x - i * a.heads;
    const int page = a.pages[i];
    if (page < 0 || page >= a.num_pages) {
        if (threadIdx.x == 0) raise_status(a.status, kPagedBadPage);
        return;
    }
    const uint8_t* const src = a.layer + (static_cast<size_t>(page) * a.heads + head) * paged_block_bytes(P, D);
    const float2 scale = *reinterpret_cast<const float2*>(src + 2 * static_cast<size_t>(P) * D);
    for (int k = threadIdx.x; k < 2 * P * kChunks; k += 256) {
        const bool second = k >= P * kChunks;
        T* const dst = static_cast<T*>(second ? a.values : a.keys);
        if (!dst) continue;
        const int j = second ? k - P * kChunks : k, t = j / kChunks, c = j % kChunks;
        float v[16];
        decode16(v, *reinterpret_cast<const uint4*>(src + (second ? static_cast<size_t>(P) * D : 0) + static_cast<size_t>(t) * D +
                                                    16 * (second ? value_chunk<D>(t, c) : key_chunk<D>(t, c))), second ? scale.y : scale.x);
        T* const to = dst + ((static_cast<size_t>(i) * P + t) * a.heads + head) * D + 16 * c;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int m = 0; m < 4; ++m) reinterpret_cast<float4*>(to)[m] = make_float4(v[4 * m], v[4 * m + 1], v[4 * m + 2], v[4 * m + 3]);
        } else {
            float lo[8], hi[8];
#pragma unroll
            for (int m = 0; m < 8; ++m) {
                lo[m] = v[m];
                hi[m] = v[8 + m];
            }
            reinterpret_cast<uint4*>(to)[0] = pack_halves(lo);
            reinterpret_cast<uint4*>(to)[1] = pack_halves(hi);
        }
    }
}

}  // namespace

void launch_paged_plan(const PagedPlanArgs& a, cudaStream_t st) {
    const long out = std::max({a.slots || a.positions ? static_cast<long>(a.tokens) : 0L, a.tables ? static_cast<long>(a.n) * a.tables_width : 0L,
                               static_cast<long>(a.tokens / a.b.page_tokens)});
    const size_t smem = (5 * static_cast<size_t>(a.n) + 3) * sizeof(int);
    static std::atomic<unsigned long long> set_all{0}, set_output{0}, set_commit{0};
    if (out <= kOneCluster) launch_cluster(paged_plan_kernel<true, true>, plan_ctas(out), true, smem, a, st, set_all);
    else {
        launch_cluster(paged_plan_kernel<true, false>, static_cast<int>(std::min<long>(a.sms, (out + kPlanThreads - 1) / kPlanThreads)), false, smem, a, st, set_output);
        launch_cluster(paged_plan_kernel<false, true>, 1, true, smem, a, st, set_commit);
    }
}
void launch_paged_truncate(const PagedPlanArgs& a, cudaStream_t st) {
    static std::atomic<unsigned long long> set{0};
    launch_cluster(paged_truncate_kernel, plan_ctas(std::min<long>(static_cast<long>(a.n) * a.b.max_pages, a.b.num_pages)), true,
                   (3 * static_cast<size_t>(a.n) + 1) * sizeof(int), a, st, set);
}
void launch_paged_init(uint8_t* layer, size_t blocks, size_t block_bytes, cudaStream_t st) {
    paged_init_kernel<<<static_cast<unsigned int>(std::min<size_t>(blocks, 4096)), 256, 0, st>>>(layer, blocks, block_bytes);
    TQ_CUDA(cudaGetLastError());
}
void launch_paged_append(const PagedAppendArgs& a, int dim, bool half, cudaStream_t st) {
    const int es = half ? 2 : 4;
    const bool wide = ((reinterpret_cast<uintptr_t>(a.keys) | reinterpret_cast<uintptr_t>(a.values) | static_cast<uintptr_t>(a.key_stride * es) |
                        static_cast<uintptr_t>(a.value_stride * es)) & 15) == 0;
    auto go = [&](auto d, auto t) {
        if (wide) launch_append_typed<d(), decltype(t), true>(a, st);
        else launch_append_typed<d(), decltype(t), false>(a, st);
    };
    using D64 = std::integral_constant<int, 64>;
    using D128 = std::integral_constant<int, 128>;
    if (dim == 64) half ? go(D64{}, __half{}) : go(D64{}, float{});
    else half ? go(D128{}, __half{}) : go(D128{}, float{});
}
void launch_paged_read(const PagedReadArgs& a, int dim, bool half, cudaStream_t st) {
    const dim3 grid(static_cast<unsigned int>(a.n) * a.heads), block(256);
    if (dim == 64) half ? launch_pdl(paged_read_kernel<64, __half>, grid, block, 0, st, a) : launch_pdl(paged_read_kernel<64, float>, grid, block, 0, st, a);
    else half ? launch_pdl(paged_read_kernel<128, __half>, grid, block, 0, st, a) : launch_pdl(paged_read_kernel<128, float>, grid, block, 0, st, a);
}

}  // namespace tq
