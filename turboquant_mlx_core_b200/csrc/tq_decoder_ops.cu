// The element-wise glue of a decoder layer around the quantised linears and the compressed-cache
// attention: RMSNorm, rotary position embedding, SwiGLU.  The reference leaves these to MLX
// (mlx::core::fast::rms_norm / rope and plain array arithmetic in the host application); they are here
// so that a whole tensor-parallel decode step can be timed.  fp16 in and out, fp32 arithmetic;
// every kernel is memory-bound (a few bytes per element) and carries the programmatic-launch wait
// so that it can follow the kernels of this library without a launch gap.
#include <algorithm>
#include <cmath>
#include <cstdint>

#include "tq_common.cuh"
#include "tq_host.hpp"
#include "tq_kernels.cuh"

namespace tq {

namespace {

__device__ __forceinline__ void ops_dependency_sync() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
}

// y[r, :] = x[r, :] * rsqrt(mean(x[r, :]^2) + eps) * w      one CTA per row
template <bool WIDE, int KEEP>
__global__ void __launch_bounds__(kRowNormThreads, row_ctas(KEEP)) rmsnorm_kernel(const __half* __restrict__ x, const __half* __restrict__ w, __half* __restrict__ y,
                                                      int cols, float eps) {
    ops_dependency_sync();
    behind_wait(x, w);
    rmsnorm_row<WIDE, KEEP>(x + static_cast<size_t>(blockIdx.x) * cols, w, y + static_cast<size_t>(blockIdx.x) * cols, cols, eps);
}

// Rotary embedding, "rotate half" convention: element i of a head pairs with element i + d/2;
// angle = position * theta^(-2 i / d).  x: [rows, heads, d] in place, positions: [rows].
// A second tensor x2 [rows, heads2, d] (the keys beside the queries) rides in the same launch: pairs beyond x's.
__global__ void __launch_bounds__(128) rope_kernel(__half* __restrict__ x, const int* __restrict__ positions, int heads, int dim,
                                                   float log2_theta, long total_pairs, __half* __restrict__ x2, int heads2, long total_pairs2) {
    ops_dependency_sync();
    behind_wait(x, positions, x2);
    const int half = dim >> 1;
    for (long i0 = static_cast<long>(blockIdx.x) * blockDim.x + threadIdx.x; i0 < total_pairs + total_pairs2;
         i0 += static_cast<long>(gridDim.x) * blockDim.x) {
        const bool second = i0 >= total_pairs;
        const long i = second ? i0 - total_pairs : i0;
        __half* const xb = second ? x2 : x;
        const int hh = second ? heads2 : heads;
        const int p = static_cast<int>(i % half);
        const long vec = i / half;               // (row, head)
        const long row = vec / hh;
        const float inv_freq = exp2f(-log2_theta * (2.0f * static_cast<float>(p) / static_cast<float>(dim)));
        float s, c;
        sincosf(static_cast<float>(positions[row]) * inv_freq, &s, &c);
        __half* v = xb + vec * dim;
        const float a = __half2float(v[p]), b = __half2float(v[p + half]);
        v[p] = __float2half_rn(a * c - b * s);
        v[p + half] = __float2half_rn(b * c + a * s);
    }
}

// The same for heads of a multiple of 16 elements, 16-byte aligned: a CTA per row.  The angles of a row are the same for all
// its heads: dim / 2 threads take the sines and cosines once, to shared memory, and a thread rotates eight pairs at a time
// (2048 rows of 28 + 4 heads of 128: 34 us with a sine and a cosine per pair and 2-byte accesses).
constexpr int kRopeThreads = 256, kRopeHalfMax = 256;
__global__ void __launch_bounds__(kRopeThreads) rope_rows_kernel(__half* __restrict__ x, const int* __restrict__ positions, int heads, int dim,
                                                                 float log2_theta, __half* __restrict__ x2, int heads2) {
    ops_dependency_sync();
    behind_wait(x, positions, x2);
    __shared__ __align__(16) float s_cos[kRopeHalfMax], s_sin[kRopeHalfMax];
    const int half = dim >> 1, per_head = half / 8, items = (heads + heads2) * per_head;
    const long row = blockIdx.x;
    for (int p = threadIdx.x; p < half; p += kRopeThreads) {
        const float inv_freq = exp2f(-log2_theta * (2.0f * static_cast<float>(p) / static_cast<float>(dim)));
        sincosf(static_cast<float>(positions[row]) * inv_freq, &s_sin[p], &s_cos[p]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < items; i += kRopeThreads) {
        const int h = i / per_head, p = (i - h * per_head) * 8;
        __half* const v = (h < heads ? x + (row * heads + h) * dim : x2 + (row * heads2 + (h - heads)) * dim) + p;
        float a[8], b[8], lo[8], hi[8];
        unpack_halves(*reinterpret_cast<const uint4*>(v), a);
        unpack_halves(*reinterpret_cast<const uint4*>(v + half), b);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float c = s_cos[p + j], s = s_sin[p + j];
            lo[j] = a[j] * c - b[j] * s;
            hi[j] = b[j] * c + a[j] * s;
        }
        *reinterpret_cast<uint4*>(v) = pack_halves(lo);
        *reinterpret_cast<uint4*>(v + half) = pack_halves(hi);
    }
}

// The norm of each query and key head and its rotation in one pass:
//
//   y = x rsqrt(mean(x^2) + eps) w,  (y_i, y_{i + D/2}) turned by position * theta^(-2 i / D)
//
// fp32 from the sum of squares to the rotation, one rounding at the end.  The angle is a fraction of a turn: position times the frequency in units
// of 2^-64 turns, of which a 64-bit product keeps the fraction without a rounding.  The frequencies come from 64-bit floats: 25 of their roundings, of
// 2^-53 of a frequency each, are 2^-51 turns at most (against 60 digits, theta 10 to 5e8 and heads of 16 to 512: 2^-54), so that the fraction is off
// by that times the position: 2^-30 turns at position 2^24, 2^-23 at 2^31, beside the 2^-26 of its rounding to 24 bits (a product in fp32 is a
// hundredth of a radian off at position 131072).
//
// A thread takes eight pairs of a head, 16 bytes from either half, so that the rotation stays in its registers, and the same pairs of the same head
// in several rows, so that it keeps the weights and finds its place once; `lanes` threads, the next power of two above D / 16, share a head and its sum
// of squares.  It is bound by memory, 16 bytes in and out for eight elements (few rows: by latency, 2.4 us replayed in a graph, as all times here): a row's values are asked for while the one
// before is at work, the first one's in front of the sines and cosines, which D / 2 threads take for all heads of a row.  8192 rows of 40 + 8 heads of
// 128: 36.5 us, 5.5 TB/s, 84 % of a plain copy's rate (52 with a row to a CTA, whose threads find head and pair anew for each 64 bytes; 44.6 with sines
// and cosines in the pairs' order, where four threads of eight read the same banks; 41.5 in 75 registers, of which two CTAs of 384 threads fill an SM
// instead of three, though heads of 64, 16 + 4 of them, take 10.4 with those and 11.3 with these).
constexpr int kHeadHalfMax = 256;
struct QkNormArgs {
    const __half* x[2];       // queries, keys
    const __half* w[2];
    __half* y[2];
    long x_stride[2], y_stride[2];   // elements from row to row
    const int* positions;
    long rows;
    int heads[2], dim, lanes;
    int width, rounds, beside, rows_each;   // threads of a row, and their rounds; rows side by side in a CTA, and one behind the other
    float eps;
    unsigned long long turns[kHeadHalfMax];   // frequencies in 2^-64 turns
};
template <bool WIDE>
__device__ __forceinline__ uint4 load_head(const __half* p) {
    if constexpr (WIDE) {
        return *reinterpret_cast<const uint4*>(p);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = __half_as_ushort(p[2 * k]) | static_cast<uint32_t>(__half_as_ushort(p[2 * k + 1])) << 16;
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
}
template <bool WIDE>
__device__ __forceinline__ void store_head(__half* p, const uint4& v) {
    if constexpr (WIDE) {
        *reinterpret_cast<uint4*>(p) = v;
    } else {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            p[2 * k] = __ushort_as_half(static_cast<unsigned short>(w[k]));
            p[2 * k + 1] = __ushort_as_half(static_cast<unsigned short>(w[k] >> 16));
        }
    }
}
template <bool WIDE>
__global__ void __maxnreg__(56) qk_norm_rope_kernel(const __grid_constant__ QkNormArgs a) {
    ops_dependency_sync();
    // [rows of the CTA][4][dim / 16][2] cosine, sine: two of a thread's pairs next to those of the next thread, which reads them beside it
    extern __shared__ __align__(16) float2 s_turn[];
    const int half = a.dim >> 1, chunks = a.dim >> 4, all = (a.heads[0] + a.heads[1]) * a.lanes, rows_cta = a.beside * a.rows_each;
    const long row0 = static_cast<long>(blockIdx.x) * rows_cta;
    const int rows = static_cast<int>(min(static_cast<long>(rows_cta), a.rows - row0));
    const int mine = a.beside > 1 ? static_cast<int>(threadIdx.x) / a.width : 0, place = static_cast<int>(threadIdx.x) - mine * a.width;
    for (int round = 0; round < a.rounds; ++round) {   // (by all threads: the barrier, the sums' shuffles)
        const int i = min(place + round * a.width, all - 1), h = i / a.lanes, t = 8 * (i - h * a.lanes), which = h >= a.heads[0] ? 1 : 0;
        const bool live = t < half && mine < a.beside && place + round * a.width < all;
        const long at = static_cast<long>(which ? h - a.heads[0] : h) * a.dim + t;
        const __half* x = a.x[which] + (row0 + mine) * a.x_stride[which] + at;
        __half* y = a.y[which] + (row0 + mine) * a.y_stride[which] + at;
        const long x_step = a.beside * a.x_stride[which], y_step = a.beside * a.y_stride[which];
        uint4 lo = make_uint4(0u, 0u, 0u, 0u), hi = lo, wl = lo, wh = lo;
        if (live && mine < rows) {
            lo = load_head<WIDE>(x);
            hi = load_head<WIDE>(x + half);
        }
        if (live) {
            wl = load_head<WIDE>(a.w[which] + t);
            wh = load_head<WIDE>(a.w[which] + t + half);
        }
        if (round == 0) {
            for (int k = threadIdx.x; k < rows * half; k += blockDim.x) {
                const int r = k / half, p = k - r * half;
                const unsigned long long turn = static_cast<unsigned long long>(static_cast<long long>(a.positions[row0 + r])) * a.turns[p];
                const float angle = static_cast<float>(static_cast<int>(turn >> 32)) * 4.656612873077393e-10f;   // half turns, -1 .. 1
                float s, c;
                sincospif(angle, &s, &c);
                s_turn[r * half + ((p >> 1 & 3) * chunks + (p >> 3)) * 2 + (p & 1)] = make_float2(c, s);
            }
            __syncthreads();
        }
        float g[8], k[8];
        unpack_halves(wl, g);
        unpack_halves(wh, k);
        for (int r = mine; r - mine < rows; r += a.beside) {   // (warps stay together: rows that are not there are zeros)
            float u[8], v[8];
            unpack_halves(lo, u);
            unpack_halves(hi, v);
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) sum = fmaf(u[j], u[j], fmaf(v[j], v[j], sum));
            __half* const to = y;
            x += x_step;
            y += y_step;
            if (live && r + a.beside < rows) {
                lo = load_head<WIDE>(x);
                hi = load_head<WIDE>(x + half);
            }
            for (int o = a.lanes >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (!live || r >= rows) continue;
            const float scale = rsqrtf(sum / static_cast<float>(a.dim) + a.eps);
            const float4* const turn = reinterpret_cast<const float4*>(s_turn + r * half) + (t >> 3);
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const float4 two = turn[(j >> 1) * chunks];
                const float p0 = u[j] * scale * g[j], q0 = v[j] * scale * k[j], p1 = u[j + 1] * scale * g[j + 1], q1 = v[j + 1] * scale * k[j + 1];
                u[j] = p0 * two.x - q0 * two.y;
                v[j] = q0 * two.x + p0 * two.y;
                u[j + 1] = p1 * two.z - q1 * two.w;
                v[j + 1] = q1 * two.z + p1 * two.w;
            }
            store_head<WIDE>(to, pack_halves(u));
            store_head<WIDE>(to + half, pack_halves(v));
        }
    }
}

// act[r, j] = silu(gate_up[r, j]) * gate_up[r, inter + j]      (gate rows first, then up rows)
__device__ __forceinline__ float swiglu(float g, float u) { return g / (1.0f + __expf(-g)) * u; }
// Rows of a multiple of eight elements, 16-byte aligned: eight per thread, a row per blockIdx.y (2048 x 18944: 77 us with
// two per thread and a 64-bit division for each pair).
__global__ void __launch_bounds__(256) swiglu_wide_kernel(const __half* __restrict__ gate_up, __half* __restrict__ act, int inter, long rows) {
    ops_dependency_sync();
    behind_wait(gate_up);
    const int j = (blockIdx.x * 256 + threadIdx.x) * 8;
    if (j >= inter) return;
    for (long r = blockIdx.y; r < rows; r += gridDim.y) {
        const __half* const src = gate_up + r * 2 * inter + j;
        float g[8], u[8];
        unpack_halves(*reinterpret_cast<const uint4*>(src), g);
        unpack_halves(*reinterpret_cast<const uint4*>(src + inter), u);
#pragma unroll
        for (int k = 0; k < 8; ++k) g[k] = swiglu(g[k], u[k]);
        *reinterpret_cast<uint4*>(act + r * inter + j) = pack_halves(g);
    }
}
__global__ void __launch_bounds__(256) swiglu_kernel(const __half* __restrict__ gate_up, __half* __restrict__ act, int inter, long rows) {
    ops_dependency_sync();
    behind_wait(gate_up);
    const long total = rows * inter;
    for (long i = (static_cast<long>(blockIdx.x) * blockDim.x + threadIdx.x) * 2; i < total; i += static_cast<long>(gridDim.x) * blockDim.x * 2) {
        const long r = i / inter, j = i - r * inter;
        const float2 g = __half22float2(*reinterpret_cast<const __half2*>(gate_up + r * 2 * inter + j));
        const float2 u = __half22float2(*reinterpret_cast<const __half2*>(gate_up + r * 2 * inter + inter + j));
        *reinterpret_cast<__half2*>(act + i) = __floats2half2_rn(swiglu(g.x, u.x), swiglu(g.y, u.y));
    }
}

cudaLaunchConfig_t ops_config(unsigned grid, unsigned block, cudaStream_t stream, cudaLaunchAttribute* attr) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cfg;
}

}  // namespace

void launch_rmsnorm_f16(const __half* x, const __half* weight, __half* y, long rows, int cols, float eps, cudaStream_t stream) {
    TQ_REQUIRE(x && weight && y, "rmsnorm: NULL argument");
    TQ_REQUIRE(cols > 0 && cols % 2 == 0, "rmsnorm: an even number of columns");
    if (rows == 0) return;
    cudaLaunchAttribute attr[1];
    cudaLaunchConfig_t cfg = ops_config(static_cast<unsigned>(rows), kRowNormThreads, stream, attr);
    decltype(&rmsnorm_kernel<true, 1>) kernel;
    TQ_ROW_KERNEL(kernel, rmsnorm_kernel, rows_wide(cols, x, weight, y), cols)
    TQ_CUDA(cudaLaunchKernelEx(&cfg, kernel, x, weight, y, cols, eps));
}

// Whether the row kernel took the call: head sizes up to 512 in sixteens, aligned tensors.
static bool launch_rope_rows(__half* x, __half* x2, const int* positions, long rows, int heads, int heads2, int dim, float theta,
                             cudaStream_t stream) {
    if (dim % 16 != 0 || dim / 2 > kRopeHalfMax || (reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(x2)) % 16 != 0 || rows >= (1L << 31) ||
        (static_cast<long>(heads) + heads2) * dim >= (1L << 31))
        return false;
    cudaLaunchAttribute attr[1];
    cudaLaunchConfig_t cfg = ops_config(static_cast<unsigned>(rows), kRopeThreads, stream, attr);
    TQ_CUDA(cudaLaunchKernelEx(&cfg, rope_rows_kernel, x, positions, heads, dim, std::log2(theta), x2, heads2));
    return true;
}

void launch_rope_f16(__half* x, const int* positions, long rows, int heads, int dim, float theta, cudaStream_t stream) {
    TQ_REQUIRE(x && positions, "rope: NULL argument");
    TQ_REQUIRE(dim > 0 && dim % 2 == 0 && heads > 0 && theta > 1.0f, "rope: bad shape");
    if (rows == 0) return;
    if (launch_rope_rows(x, nullptr, positions, rows, heads, 0, dim, theta, stream)) return;
    const long pairs = rows * heads * (dim / 2);
    long blocks = (pairs + 127) / 128;
    if (blocks > 1184) blocks = 1184;
    cudaLaunchAttribute attr[1];
    cudaLaunchConfig_t cfg = ops_config(static_cast<unsigned>(blocks), 128, stream, attr);
    TQ_CUDA(cudaLaunchKernelEx(&cfg, rope_kernel, x, positions, heads, dim, std::log2(theta), pairs, static_cast<__half*>(nullptr), 1, 0L));
}

void launch_rope_qk_f16(__half* q, __half* k, const int* positions, long rows, int q_heads, int kv_heads, int dim, float theta,
                        cudaStream_t stream) {
    TQ_REQUIRE(q && k && positions, "rope: NULL argument");
    TQ_REQUIRE(dim > 0 && dim % 2 == 0 && q_heads > 0 && kv_heads > 0 && theta > 1.0f, "rope: bad shape");
    if (rows == 0) return;
    if (launch_rope_rows(q, k, positions, rows, q_heads, kv_heads, dim, theta, stream)) return;
    const long pairs_q = rows * q_heads * (dim / 2), pairs_k = rows * kv_heads * (dim / 2);
    long blocks = (pairs_q + pairs_k + 127) / 128;
    if (blocks > 1184) blocks = 1184;
    cudaLaunchAttribute attr[1];
    cudaLaunchConfig_t cfg = ops_config(static_cast<unsigned>(blocks), 128, stream, attr);
    TQ_CUDA(cudaLaunchKernelEx(&cfg, rope_kernel, q, positions, q_heads, dim, std::log2(theta), pairs_q, k, kv_heads, pairs_k));
}

void launch_qk_norm_rope_f16(const __half* q, const __half* k, const __half* q_weight, const __half* k_weight, const int* positions, long rows, int q_heads,
                             int kv_heads, int dim, long q_stride, long k_stride, float eps, float theta, __half* q_out, __half* k_out, long q_out_stride,
                             long k_out_stride, cudaStream_t stream) {
    QkNormArgs a{};
    a.x[0] = q;
    a.x[1] = k;
    a.w[0] = q_weight;
    a.w[1] = k_weight;
    a.y[0] = q_out;
    a.y[1] = k_out;
    a.x_stride[0] = q_stride;
    a.x_stride[1] = k_stride;
    a.y_stride[0] = q_out_stride;
    a.y_stride[1] = k_out_stride;
    a.positions = positions;
    a.rows = rows;
    a.heads[0] = q_heads;
    a.heads[1] = kv_heads;
    a.dim = dim;
    a.eps = eps;
    a.lanes = 1;
    while (a.lanes * 16 < dim) a.lanes *= 2;
    constexpr double kTwoPi = 6.283185307179586476925286766559;
    // (a power for every eighth, the others up to seven products of it, 25 2^-53 off in all, where a power each took two thirds of the call)
    const double ratio = std::pow(static_cast<double>(theta), -2.0 / dim);
    for (int i = 0; i < dim / 2; i += 8) {
        double turn = std::pow(static_cast<double>(theta), -2.0 * i / dim) / kTwoPi * 18446744073709551616.0;
        for (int k = i; k < i + 8; ++k, turn *= ratio) a.turns[k] = static_cast<unsigned long long>(std::llrint(turn));
    }
    uintptr_t all = 0;
    for (int i = 0; i < 2; ++i)
        all |= reinterpret_cast<uintptr_t>(a.x[i]) | reinterpret_cast<uintptr_t>(a.w[i]) | reinterpret_cast<uintptr_t>(a.y[i]) | static_cast<uintptr_t>(2 * (a.x_stride[i] | a.y_stride[i]));
    // Threads of a row (in several rounds above 512, then of whole warps); rows side by side where a row has few, and as many behind one another, up to
    // four, as leave four CTAs to each SM.
    const int per_row = (q_heads + kv_heads) * a.lanes;
    a.rounds = (per_row + 511) / 512;
    a.width = a.rounds == 1 ? per_row : ((per_row + a.rounds - 1) / a.rounds + 31) / 32 * 32;
    a.beside = static_cast<int>(std::min<long>(std::max(1, 256 / a.width), rows));
    a.rows_each = static_cast<int>(std::min<long>(4, std::max<long>(1, rows / (a.beside * 4L * sm_count(current_device())))));
    const int rows_cta = a.beside * a.rows_each, threads = (a.beside * a.width + 31) / 32 * 32;
    const dim3 grid(static_cast<unsigned>((rows + rows_cta - 1) / rows_cta)), block(static_cast<unsigned>(threads));
    const size_t smem = static_cast<size_t>(rows_cta) * (dim / 2) * sizeof(float2);
    if (all % 16 == 0) launch_pdl(qk_norm_rope_kernel<true>, grid, block, smem, stream, a);
    else launch_pdl(qk_norm_rope_kernel<false>, grid, block, smem, stream, a);
}

void launch_swiglu_f16(const __half* gate_up, __half* act, long rows, int inter, cudaStream_t stream) {
    TQ_REQUIRE(gate_up && act, "swiglu: NULL argument");
    TQ_REQUIRE(inter > 0 && inter % 2 == 0, "swiglu: an even intermediate size");
    if (rows == 0) return;
    cudaLaunchAttribute attr[1];
    if (inter % 8 == 0 && (reinterpret_cast<uintptr_t>(gate_up) | reinterpret_cast<uintptr_t>(act)) % 16 == 0) {
        cudaLaunchConfig_t wide = ops_config(static_cast<unsigned>((inter / 8 + 255) / 256), 256, stream, attr);
        wide.gridDim.y = static_cast<unsigned>(rows < 65535 ? rows : 65535);
        TQ_CUDA(cudaLaunchKernelEx(&wide, swiglu_wide_kernel, gate_up, act, inter, rows));
        return;
    }
    long blocks = (rows * inter / 2 + 255) / 256;
    if (blocks > 1184) blocks = 1184;
    cudaLaunchConfig_t cfg = ops_config(static_cast<unsigned>(blocks), 256, stream, attr);
    TQ_CUDA(cudaLaunchKernelEx(&cfg, swiglu_kernel, gate_up, act, inter, rows));
}

}  // namespace tq
