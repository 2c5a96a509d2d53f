// C entry points of a drafted decoding step that belong to no cache: the norms of heads with their rotation, and the verification of drafts.  The
// reference leaves both to its host application.
#include <cmath>

#include "tq_drafts.cuh"
#include "tq_host.hpp"
#include "tq_kernels.cuh"
#include "turboquant_c/turboquant_b200.h"

using namespace tq;

namespace {
// The device of the call's memory is current in here, and the caller's again behind.
class OnDevice {
public:
    explicit OnDevice(const void* p) {
        cudaPointerAttributes attr{};
        TQ_CUDA(cudaPointerGetAttributes(&attr, p));
        TQ_CUDA(cudaGetDevice(&before_));
        if (attr.device != before_) {
            TQ_CUDA(cudaSetDevice(attr.device));
            moved_ = true;
        }
    }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;
    ~OnDevice() {
        if (moved_) cudaSetDevice(before_);
    }

private:
    int before_ = 0;
    bool moved_ = false;
};
}  // namespace

extern "C" {

int tq_qk_norm_rope_f16(const void* q_fp16, const void* k_fp16, const void* q_weight_fp16, const void* k_weight_fp16, const int* positions, long rows,
                        int q_heads, int kv_heads, int head_dim, long q_stride, long k_stride, float eps, float theta, void* q_out_fp16, void* k_out_fp16,
                        long q_out_stride, long k_out_stride, void* stream) {
    return guarded<int>(0, -1, [&]() {
        TQ_REQUIRE(rows >= 0 && rows < (1L << 31), "qk norm: bad number of rows");
        TQ_REQUIRE(q_heads > 0 && kv_heads > 0 && q_heads <= 65536 && kv_heads <= 65536, "qk norm: 1 to 65536 heads each");
        TQ_REQUIRE(head_dim > 0 && head_dim <= 512 && head_dim % 16 == 0, "qk norm: head_dim must be a multiple of 16, up to 512");
        TQ_REQUIRE(std::isfinite(theta) && theta > 1.f, "qk norm: theta must be finite and above 1");
        TQ_REQUIRE(std::isfinite(eps) && eps >= 0.f, "qk norm: eps must be finite and not negative");
        const long q_row = static_cast<long>(q_heads) * head_dim, k_row = static_cast<long>(kv_heads) * head_dim;
        TQ_REQUIRE(q_stride >= q_row && q_out_stride >= q_row && k_stride >= k_row && k_out_stride >= k_row, "qk norm: a row's stride is shorter than its heads");
        if (rows == 0) return 0;
        for (const void* p : {q_fp16, k_fp16, q_weight_fp16, k_weight_fp16, static_cast<const void*>(positions), static_cast<const void*>(q_out_fp16),
                              static_cast<const void*>(k_out_fp16)})
            TQ_REQUIRE(is_device_pointer(p), "qk norm: arguments must be device pointers");
        // (in place each thread writes what it alone has read; anywhere else over an argument another CTA may not have read it yet)
        const ByteRows in[] = {{q_fp16, 2ul * q_row, rows, 2ul * q_stride}, {k_fp16, 2ul * k_row, rows, 2ul * k_stride}, {q_weight_fp16, 2ul * head_dim},
                               {k_weight_fp16, 2ul * head_dim}, {positions, 4ul * rows}};
        const ByteRows out[] = {{q_out_fp16, 2ul * q_row, rows, 2ul * q_out_stride}, {k_out_fp16, 2ul * k_row, rows, 2ul * k_out_stride}};
        for (int i = 0; i < 2; ++i)
            for (int j = 0; j < 5; ++j)
                TQ_REQUIRE((i == j && out[i].p == in[j].p && (rows == 1 || out[i].stride == in[j].stride)) || rows_apart(out[i], in[j]),
                           "qk norm: results must be where their rows are, with the same stride, or not where an argument is");
        TQ_REQUIRE(rows_apart(out[0], out[1]), "qk norm: the two results must not be in the same place");
        const OnDevice on(q_fp16);
        const auto half = [](const void* p) { return static_cast<const __half*>(p); };
        launch_qk_norm_rope_f16(half(q_fp16), half(k_fp16), half(q_weight_fp16), half(k_weight_fp16), positions, rows, q_heads, kv_heads, head_dim, q_stride,
                                k_stride, eps, theta, static_cast<__half*>(q_out_fp16), static_cast<__half*>(k_out_fp16), q_out_stride, k_out_stride,
                                static_cast<cudaStream_t>(stream));
        return 0;
    });
}

int tq_verify_drafts(const int* starts, const int* parents, const int* tokens, int n, int rows, const void* target, const void* draft, int dtype, int vocab,
                     long target_stride, long draft_stride, const float* uniforms, int* path, int width, int* kept, int* next, void* stream) {
    return guarded<int>(0, -1, [&]() {
        TQ_REQUIRE(n >= 0 && n <= 65536 && rows >= 0, "verify drafts: bad number of requests or rows");
        TQ_REQUIRE(vocab > 0 && vocab <= kDraftVocab, "verify drafts: a vocabulary has 1 to " + std::to_string(kDraftVocab) + " tokens");
        TQ_REQUIRE(width > 0, "verify drafts: a path has room for one node at least");
        TQ_REQUIRE(dtype == TQ_F32 || dtype == TQ_F16, "verify drafts: probabilities must be fp32 or fp16");
        TQ_REQUIRE(target_stride >= vocab && (!draft || draft_stride >= vocab), "verify drafts: a row's stride is shorter than the vocabulary");
        if (n == 0) return 0;
        for (const void* p : {static_cast<const void*>(starts), static_cast<const void*>(path), static_cast<const void*>(kept), static_cast<const void*>(next)})
            TQ_REQUIRE(is_device_pointer(p), "verify drafts: arguments must be device pointers");
        for (const void* p : {static_cast<const void*>(parents), static_cast<const void*>(tokens), target, static_cast<const void*>(uniforms)})
            TQ_REQUIRE(rows == 0 || is_device_pointer(p), "verify drafts: arguments must be device pointers");
        TQ_REQUIRE(rows == 0 || !draft || is_device_pointer(draft), "verify drafts: arguments must be device pointers");
        // (the CTAs of a request read what they decide by in their own time, and must all see the same)
        const size_t es = dtype == TQ_F16 ? 2 : 4;
        const ByteRows all[] = {{path, 4ul * n * width}, {kept, 4ul * n}, {next, 4ul * n}, {starts, 4ul * n + 4}, {parents, 4ul * rows}, {tokens, 4ul * rows},
                                {uniforms, 4ul * rows}, {target, vocab * es, rows, target_stride * es}, {draft, vocab * es, draft ? rows : 0, draft_stride * es}};
        for (int i = 0; i < 3; ++i)
            for (int j = i + 1; j < 9; ++j) TQ_REQUIRE(rows_apart(all[i], all[j]), "verify drafts: results must not be where an argument or another result is");
        const OnDevice on(starts);
        launch_verify_drafts({starts, parents, tokens, target, draft, uniforms, target_stride, draft ? draft_stride : 0, rows, vocab, width, 0, path, kept, next}, n,
                             dtype == TQ_F16, static_cast<cudaStream_t>(stream));
        return 0;
    });
}

}  // extern "C"
