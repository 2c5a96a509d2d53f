// Which drafted tokens stay: a walk down each request's tree of drafts that tests the children of the present node against the target's
// probabilities, with the caller's random numbers, and the token that follows.
//
// p is the target's row of the present node, q the draft's.  The children's tokens were drawn from q, one after another, and each one is accepted where
//
//   u Z q(x) < w(x),   w = max(p - S q, 0),  Z = sum of w        (S = 0, Z = 1 at first; a rejection adds Z to S)
//
// which is what is left of p after the rejections, max(max(p - Z0 q, 0) - Z1 q, 0) = max(p - (Z0 + Z1) q, 0), so that one number stands
// for them all.  Where no child is accepted the next token is drawn from w.  Either way each token is distributed as the target's rows have it.
// Without q the children are points: accepted where u Z < w(x); a rejection takes w(x) off Z and x out of w.
//
// A request has a cluster of CTAs, each of them a part of the vocabulary.  All of them make the walk, from what thread j looks up for node j in
// advance (its token's two probabilities in its parent's rows), so that a test is a few reads of shared memory; only a rejection with q, and the
// end, need a pass over rows: a warp sums a contiguous part, the warps' sums go to all CTAs of the cluster, and each adds them up in the same
// order.  The warp in whose part the sum passes u0 Z goes over it once more.  Sums, products and comparisons are in 64 bits: a token is a whole
// number, and a comparison of sums in 32 bits would go wrong next to a border, of which there are as many as tokens.
//
// What bounds it: latency.  Few requests: three loads behind one another, a pass, the cluster's barriers, the last part once more, 10 us for one (as all
// times here, replayed in a graph).  Many: the request that takes most passes, each of them some rounds of loads, sums in 64 bits and a barrier of the
// cluster: 64 requests of 16 nodes in 39 us, 3 TB/s of rows out of memory and L2 cache, with a third of the issue slots and a sixth of the conversions' rate in use.

#include <cooperative_groups.h>

#include <algorithm>
#include <cstdint>

#include "tq_drafts.cuh"

namespace tq {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512, kWarps = kThreads / 32, kMaxCtas = 8;
constexpr int kAtOnce = 2;   // 16-byte pieces of a row that a lane asks for at once (four, and one CTA to an SM: 52 us instead of 39 below)

template <typename T>
__device__ __forceinline__ float probability(const T* row, int x) {
    const float p = static_cast<float>(row[x]);
    return p > 0.f ? p : 0.f;   // (NaN too)
}

// 16 bytes of a row, elements e and on; zeros beyond its end.
template <typename T, bool WIDE>
__device__ __forceinline__ uint4 load_row(const T* row, int e, int end) {
    constexpr int VEC = 16 / sizeof(T);
    if (WIDE && e + VEC <= end) return *reinterpret_cast<const uint4*>(row + e);
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if constexpr (sizeof(T) == 4) {
            w[k] = e + k < end ? __float_as_uint(row[e + k]) : 0u;
        } else {
            const uint32_t lo = e + 2 * k < end ? __half_as_ushort(row[e + 2 * k]) : 0u, hi = e + 2 * k + 1 < end ? __half_as_ushort(row[e + 2 * k + 1]) : 0u;
            w[k] = lo | hi << 16;
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// They as numbers, 0 for what is no positive one.
template <typename T>
__device__ __forceinline__ void numbers(float (&v)[16 / sizeof(T)], const uint4& raw) {
    if constexpr (sizeof(T) == 2) {
        unpack_halves(raw, v);
    } else {
        v[0] = __uint_as_float(raw.x);
        v[1] = __uint_as_float(raw.y);
        v[2] = __uint_as_float(raw.z);
        v[3] = __uint_as_float(raw.w);
    }
#pragma unroll
    for (int k = 0; k < static_cast<int>(16 / sizeof(T)); ++k) v[k] = v[k] > 0.f ? v[k] : 0.f;
}

// The parts' sums, four (or fewer) to a lane, in the lanes' order: the lane's and all in front of it.
struct PartSums {
    double each[kMaxCtas * kWarps / 32], upto, total;
    __device__ __forceinline__ void load(const double* sums, int parts, int lane) {
        constexpr int kEach = kMaxCtas * kWarps / 32;
        const int per = (parts + 31) / 32;
        upto = 0.;
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            each[k] = k < per && lane * per + k < parts ? sums[lane * per + k] : 0.;
            upto += each[k];
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double t = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += t;
        }
        total = __shfl_sync(0xffffffffu, upto, 31);
    }
};

template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads, 2) verify_kernel(const __grid_constant__ VerifyArgs a) {
    constexpr int VEC = 16 / sizeof(T), kGroup = 32 * VEC;
    pdl_wait_release();
    extern __shared__ uint32_t s_gone[];   // without q: tokens of this CTA's part of the vocabulary that were rejected, a bit each
    __shared__ int s_parent[kDraftNodes], s_token[kDraftNodes];
    __shared__ float s_u[kDraftNodes], s_p[kDraftNodes], s_q[kDraftNodes];   // a node's random number, its token's probabilities at its parent
    __shared__ double s_sum[2][kMaxCtas * kWarps];                           // of the parts, pass by pass
    __shared__ int s_path[kDraftNodes], s_list[kDraftNodes];                 // rejected tokens at the present node
    __shared__ int s_now, s_kept, s_rejected, s_again;
    __shared__ double s_subtract;

    const cg::cluster_group cluster = cg::this_cluster();
    const int ctas = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank()), i = blockIdx.x / ctas;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    cluster.barrier_arrive();
    const bool drawn = a.draft != nullptr;
    const int start = a.starts[i], end = a.starts[i + 1];
    // (a request without nodes, or one that is not inside the rows, has none)
    const int count = start >= 0 && end <= a.rows && end > start ? min(end - start, kDraftNodes) : 0;
    if (count == 0) {
        if (rank == 0) {
            for (int k = tid; k < a.width; k += kThreads) a.path[static_cast<long>(i) * a.width + k] = -1;
            if (tid == 0) {
                a.kept[i] = 0;
                a.next[i] = -1;
            }
        }
        cluster.barrier_wait();
        return;   // (the whole cluster)
    }
    const T* const target = static_cast<const T*>(a.target) + start * a.target_stride;
    const T* const draft = drawn ? static_cast<const T*>(a.draft) + start * a.draft_stride : nullptr;
    for (int j = tid; j < count; j += kThreads) {
        const int parent = a.parents[start + j], x = a.tokens[start + j];
        // (a node that has no parent in front of it, or no token, is nobody's child)
        const bool node = j > 0 && parent >= 0 && parent < j && x >= 0 && x < a.vocab;
        s_parent[j] = node ? parent : -1;
        s_token[j] = x;
        s_u[j] = a.uniforms[start + j];
        s_p[j] = node ? probability(target + parent * a.target_stride, x) : 0.f;
        s_q[j] = node && drawn ? probability(draft + parent * a.draft_stride, x) : 0.f;
    }
    const int words = (a.segment * kWarps + 31) / 32;
    if (!drawn)
        for (int k = tid; k < words; k += kThreads) s_gone[k] = 0u;
    __syncthreads();
    cluster.barrier_wait();   // every CTA of it runs: its shared memory may be written

    const int mine0 = (rank * kWarps + warp) * a.segment;   // this warp's part of the vocabulary
    int now = 0, at = 1, kept = 1, rejected = 0, turn = 0;
    double subtract = 0., left = 1.;
    if (tid == 0) s_path[0] = 0;
    // The sum of this warp's part of w = max(p - s q, 0) (without q: of p, but for tokens that are gone).
    auto part_sum = [&](const T* p_row, const T* q_row, double s, bool gaps) {
        double sum = 0.;
        const int part_end = min(mine0 + a.segment, a.vocab);
        for (int e0 = mine0; e0 < part_end; e0 += kAtOnce * kGroup) {
            uint4 p[kAtOnce], q[kAtOnce];
#pragma unroll
            for (int b = 0; b < kAtOnce; ++b) {
                const int e = e0 + b * kGroup + lane * VEC;
                p[b] = load_row<T, WIDE>(p_row, e, part_end);
                if (q_row) q[b] = load_row<T, WIDE>(q_row, e, part_end);
            }
#pragma unroll
            for (int b = 0; b < kAtOnce; ++b) {
                const int at = e0 + b * kGroup + lane * VEC - rank * kWarps * a.segment;
                const uint32_t gone = gaps && at < kWarps * a.segment ? s_gone[at >> 5] >> (at & 31) : 0u;
                float v[VEC], u[VEC];
                numbers<T>(v, p[b]);
                if (q_row) {
                    numbers<T>(u, q[b]);
#pragma unroll
                    for (int k = 0; k < VEC; ++k) sum += fmax(static_cast<double>(v[k]) - s * u[k], 0.);
                } else {
#pragma unroll
                    for (int k = 0; k < VEC; ++k) sum += gone >> k & 1u ? 0. : static_cast<double>(v[k]);
                }
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        return sum;
    };
    bool fresh = true, over = false;   // no rejection at this node; the walk is over
    double total = 0.;
    for (;;) {
        // ---- the walk, by the first warp of each CTA, up to the next pass ----
        if (warp == 0) {
            bool pass = false;
            while (!pass) {
                int child = -1;
                if (kept < a.width)
                    for (int base = at; base < count; base += 32) {
                        const unsigned int hits = __ballot_sync(0xffffffffu, base + lane < count && s_parent[base + lane] == now);
                        if (hits) {
                            child = base + __ffs(static_cast<int>(hits)) - 1;
                            break;
                        }
                    }
                if (child < 0) {
                    over = pass = true;
                    break;
                }
                at = child + 1;
                bool accepted;
                double w;
                if (drawn) {
                    const double q = s_q[child];
                    w = fmax(static_cast<double>(s_p[child]) - subtract * q, 0.);
                    accepted = static_cast<double>(s_u[child]) * left * q < w;
                } else {
                    bool again = false;
                    for (int k = lane; k < rejected; k += 32) again = again || s_list[k] == s_token[child];
                    w = __any_sync(0xffffffffu, again) ? 0. : s_p[child];
                    accepted = static_cast<double>(s_u[child]) * left < w;
                }
                if (accepted) {
                    now = child;
                    if (lane == 0) s_path[kept] = child;
                    ++kept;
                    subtract = 0.;
                    left = 1.;
                    rejected = 0;
                    fresh = true;
                } else if (drawn) {
                    subtract += left;
                    fresh = false;
                    pass = true;
                } else {
                    left -= w;
                    if (lane == 0) s_list[rejected] = s_token[child];
                    ++rejected;
                }
                __syncwarp();
            }
            if (lane == 0) {
                s_now = now;
                s_kept = kept;
                s_rejected = rejected;
                s_subtract = subtract;
                s_again = over ? (drawn && !fresh ? 2 : 1) : 0;
            }
        }
        __syncthreads();
        // (over behind a rejection: that one's sums are those of what is left)
        const int state = s_again;
        if (state == 2) break;
        if (!drawn) {
            for (int k = tid; k < s_rejected; k += kThreads) {
                const int x = s_list[k] - rank * kWarps * a.segment;
                if (x >= 0 && x < kWarps * a.segment) atomicOr(&s_gone[x >> 5], 1u << (x & 31));
            }
            __syncthreads();
        }
        const T* const p_row = target + s_now * a.target_stride;
        const T* const q_row = drawn && s_subtract > 0. ? draft + s_now * a.draft_stride : nullptr;
        const double s = s_subtract;
        const double sum = part_sum(p_row, q_row, s, !drawn);
        if (lane < ctas) *cluster.map_shared_rank(&s_sum[turn & 1][rank * kWarps + warp], lane) = sum;
        cluster.sync();
        PartSums parts;
        parts.load(s_sum[turn & 1], ctas * kWarps, lane);
        total = parts.total;
        ++turn;
        left = total;
        if (state == 1) break;
    }
    // ---- the next token ----
    const double u = s_u[0];
    const int last_turn = (turn - 1) & 1;
    now = s_now;
    double s = s_subtract;
    bool whole = false;
    if (!(total > 0.)) {
        // Nothing is left (a target that its draft covers but for roundings): the target's row as it is.
        whole = true;
        s = 0.;
        const double sum = part_sum(target + now * a.target_stride, nullptr, 0., false);
        if (lane < ctas) *cluster.map_shared_rank(&s_sum[last_turn ^ 1][rank * kWarps + warp], lane) = sum;
        cluster.sync();
    }
    PartSums parts;
    parts.load(s_sum[whole ? last_turn ^ 1 : last_turn], ctas * kWarps, lane);
    // the part in which the sum passes u total: the last one with anything where none does
    const double limit = u * parts.total;
    int owner = -1;
    double before = 0.;
    {
        constexpr int kEach = kMaxCtas * kWarps / 32;
        const int per = (ctas * kWarps + 31) / 32;
        int last = -1, passing = -1;   // of the lane's parts
        double at[kEach], upto = __shfl_up_sync(0xffffffffu, parts.upto, 1);
        if (lane == 0) upto = 0.;
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            at[k] = upto;
            upto += parts.each[k];
            if (parts.each[k] > 0.) {
                last = k;
                if (passing < 0 && upto > limit) passing = k;
            }
        }
        const unsigned int some = __ballot_sync(0xffffffffu, last >= 0), beyond = __ballot_sync(0xffffffffu, passing >= 0);
        const int src = beyond ? __ffs(static_cast<int>(beyond)) - 1 : some ? 31 - __clz(static_cast<int>(some)) : 0;
        const int k = __shfl_sync(0xffffffffu, beyond ? passing : last, src);
        if (some) owner = src * per + k;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (i == k) before = at[i];
        before = __shfl_sync(0xffffffffu, before, src);
    }
    if (rank == 0) {
        for (int k = tid; k < a.width; k += kThreads) a.path[static_cast<long>(i) * a.width + k] = k < s_kept ? s_path[k] : -1;
        if (tid == 0) {
            a.kept[i] = s_kept;
            if (owner < 0) a.next[i] = -1;
        }
    }
    if (owner != rank * kWarps + warp) return;
    int found = -1, positive = -1;   // the token; the last one so far that could be
    double sum = before;
    const int part_end = min(mine0 + a.segment, a.vocab);
    for (int e0 = mine0; found < 0 && e0 < part_end; e0 += kAtOnce * kGroup) {
        uint4 p[kAtOnce], q[kAtOnce];
#pragma unroll
        for (int b = 0; b < kAtOnce; ++b) {
            const int e = e0 + b * kGroup + lane * VEC;
            p[b] = load_row<T, WIDE>(target + now * a.target_stride, e, part_end);
            if (s > 0.) q[b] = load_row<T, WIDE>(draft + now * a.draft_stride, e, part_end);
        }
        auto weights = [&](double (&w)[VEC], int b) {
            float v[VEC], u[VEC];
            numbers<T>(v, p[b]);
            if (s > 0.) {
                numbers<T>(u, q[b]);
#pragma unroll
                for (int k = 0; k < VEC; ++k) w[k] = fmax(static_cast<double>(v[k]) - s * u[k], 0.);
            } else {
                const int at = e0 + b * kGroup + lane * VEC - rank * kWarps * a.segment;
                const uint32_t gone = !drawn && !whole && at < kWarps * a.segment ? s_gone[at >> 5] >> (at & 31) : 0u;
#pragma unroll
                for (int k = 0; k < VEC; ++k) w[k] = gone >> k & 1u ? 0. : static_cast<double>(v[k]);
            }
        };
        double own[kAtOnce], upto[kAtOnce];
#pragma unroll
        for (int b = 0; b < kAtOnce; ++b) {
            double w[VEC];
            weights(w, b);
            own[b] = 0.;
#pragma unroll
            for (int k = 0; k < VEC; ++k) own[b] += w[k];
            upto[b] = own[b];
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1)
#pragma unroll
            for (int b = 0; b < kAtOnce; ++b) {
                const double t = __shfl_up_sync(0xffffffffu, upto[b], o);
                if (lane >= o) upto[b] += t;
            }
#pragma unroll
        for (int b = 0; b < kAtOnce; ++b) {
            if (found >= 0) continue;
            const unsigned int some = __ballot_sync(0xffffffffu, own[b] > 0.), beyond = __ballot_sync(0xffffffffu, own[b] > 0. && sum + upto[b] > limit);
            int token = -1, last = -1;
            double running = sum + (upto[b] - own[b]), w[VEC];
            weights(w, b);
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                running += w[k];
                if (w[k] > 0.) {
                    last = e0 + b * kGroup + lane * VEC + k;
                    if (token < 0 && running > limit) token = last;
                }
            }
            if (token < 0) token = last;   // (the lane's own sum rounded otherwise)
            if (beyond) found = __shfl_sync(0xffffffffu, token, __ffs(static_cast<int>(beyond)) - 1);
            else if (some) positive = __shfl_sync(0xffffffffu, last, 31 - __clz(static_cast<int>(some)));
            sum += __shfl_sync(0xffffffffu, upto[b], 31);
        }
    }
    if (lane == 0) a.next[i] = found >= 0 ? found : positive;
}

}  // namespace

void launch_verify_drafts(VerifyArgs a, int n, bool half, cudaStream_t st) {
    if (n == 0) return;
    const int es = half ? 2 : 4, group = 32 * 16 / es;
    // CTAs to a request: as many as there are pieces for, up to 8 (the portable most), however many requests there are: they take one to many passes, and
    // the ones behind fill up (64 requests of 16 nodes, 151936 tokens: 39 us; with two CTAs each, which run all at once, 56, with four 44).
    int ctas = 1;
    while (ctas < kMaxCtas && ctas * kWarps * group < a.vocab) ctas *= 2;
    a.segment = ((a.vocab + ctas * kWarps - 1) / (ctas * kWarps) + group - 1) / group * group;
    uintptr_t all = reinterpret_cast<uintptr_t>(a.target) | static_cast<uintptr_t>(a.target_stride * es);
    if (a.draft) all |= reinterpret_cast<uintptr_t>(a.draft) | static_cast<uintptr_t>(a.draft_stride * es);
    const size_t smem = a.draft ? 0 : static_cast<size_t>((a.segment * kWarps + 31) / 32) * 4;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned int>(ctas);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned int>(n) * ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const auto go = [&](auto kernel) { TQ_CUDA(cudaLaunchKernelEx(&cfg, kernel, a)); };
    if (half) all % 16 == 0 ? go(verify_kernel<__half, true>) : go(verify_kernel<__half, false>);
    else all % 16 == 0 ? go(verify_kernel<float, true>) : go(verify_kernel<float, false>);
}

}  // namespace tq
