// C-ABI of the paged 8-bit KV cache (include/turboquant_c/turboquant_b200.h, tq_paged_*).  The reference's cache holds one
// sequence (include/turboquant/kv_cache.h:42-133); this one is what a server keeps beside it for the requests of a batch.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <memory>
#include <vector>

#include "tq_host.hpp"
#include "tq_paged.cuh"
#include "turboquant_c/turboquant_b200.h"

namespace turboquant {

using tq::DeviceBuffer;

class PagedKVCache {
public:
    PagedKVCache(int layers, int heads, int dim, int pages, int page_tokens, int max_requests, int max_pages, int max_tokens)
        : heads_(heads), dim_(dim), max_tokens_(max_tokens) {
        TQ_REQUIRE(layers > 0 && heads > 0 && pages > 0, "paged cache: layers, heads and pages must be positive");
        TQ_REQUIRE(heads <= 65536, "paged cache: at most 65536 heads");   // (the kernels count requests times heads in 32 bits)
        TQ_REQUIRE(dim == 64 || dim == 128, "paged cache: head_dim must be 64 or 128");
        TQ_REQUIRE(page_tokens == 16 || page_tokens == 32 || page_tokens == 64 || page_tokens == 128, "paged cache: a page holds 16, 32, 64 or 128 tokens");
        TQ_REQUIRE(max_requests > 0 && max_requests <= tq::kPagedMaxRequests, "paged cache: max_requests must be 1 .. " + std::to_string(tq::kPagedMaxRequests));
        TQ_REQUIRE(max_pages > 0 && max_tokens > 0, "paged cache: max_pages_per_request and max_tokens must be positive");
        constexpr long kMost = 1l << 30;
        TQ_REQUIRE(static_cast<long>(pages) * page_tokens <= kMost && static_cast<long>(max_pages) * page_tokens <= kMost && max_tokens <= kMost,
                   "paged cache: at most 2^30 tokens");
        TQ_REQUIRE(static_cast<long>(pages) * heads <= kMost, "paged cache: at most 2^30 pages times heads");
        device_ = tq::current_device();
        sms_ = tq::sm_count(device_);
        b_.max_requests = max_requests;
        numbers_.resize(static_cast<size_t>(max_requests));
        b_.max_pages = max_pages;
        b_.num_pages = pages;
        b_.page_tokens = page_tokens;
        b_.max_pieces = static_cast<int>(std::min<long>(max_tokens, max_tokens / page_tokens + 2l * max_requests));
        const size_t block = tq::paged_block_bytes(page_tokens, dim), blocks = static_cast<size_t>(pages) * heads;
        for (int i = 0; i < layers; ++i) {
            layers_.emplace_back();
            layers_.back().owned_by(&use_);
            layers_.back().resize(blocks * block);
            tq::launch_paged_init(layers_.back().as<uint8_t>(), blocks, block, nullptr);
        }
        // the arrays of a plan, 256-byte aligned in one block
        const size_t sizes[] = {sizeof(tq::PagedHeader), 4ul * max_requests, 4ul * max_requests * max_pages, 4ul * pages, 4ul * max_requests,
                                4ul * max_requests + 4, 4ul * max_requests, sizeof(tq::PagedPiece) * b_.max_pieces, 8ul * max_requests,
                                sizeof(tq::PagedNode) * max_tokens, sizeof(uint8_t*) * layers};
        constexpr int kArrays = sizeof(sizes) / sizeof(sizes[0]);
        size_t at[kArrays], all = 0;
        for (int i = 0; i < kArrays; ++i) {
            at[i] = all;
            all += (sizes[i] + 255) / 256 * 256;
        }
        state_.owned_by(&use_);
        state_.resize(all);
        char* const p = state_.as<char>();
        b_.header = reinterpret_cast<tq::PagedHeader*>(p + at[0]);
        b_.lengths = reinterpret_cast<int*>(p + at[1]);
        b_.tables = reinterpret_cast<int*>(p + at[2]);
        b_.stack = reinterpret_cast<int*>(p + at[3]);
        b_.rows = reinterpret_cast<int*>(p + at[4]);
        b_.starts = reinterpret_cast<int*>(p + at[5]);
        b_.held = reinterpret_cast<int*>(p + at[6]);
        b_.pieces = reinterpret_cast<tq::PagedPiece*>(p + at[7]);
        staged_ = reinterpret_cast<int*>(p + at[8]);
        b_.nodes = reinterpret_cast<tq::PagedNode*>(p + at[9]);
        b_.layers = reinterpret_cast<uint8_t* const*>(p + at[10]);
        TQ_CUDA(cudaMemset(p, 0, all));
        std::vector<uint8_t*> bases;
        for (const DeviceBuffer& l : layers_) bases.push_back(l.as<uint8_t>());
        TQ_CUDA(cudaMemcpy(p + at[10], bases.data(), sizeof(uint8_t*) * bases.size(), cudaMemcpyHostToDevice));
        std::vector<int> stack(static_cast<size_t>(pages));
        for (int i = 0; i < pages; ++i) stack[static_cast<size_t>(i)] = pages - 1 - i;   // page 0 is the first to go
        TQ_CUDA(cudaMemcpy(b_.stack, stack.data(), 4ul * pages, cudaMemcpyHostToDevice));
        TQ_CUDA(cudaMemcpy(&b_.header->free_pages, &pages, 4, cudaMemcpyHostToDevice));
        scratch_.owned_by(&use_);
        prompt_scratch_ = (tq::paged_attn_scratch_bytes(dim, sms_) + 255) / 256 * 256;   // (behind the other kernel's)
        scratch_.resize(prompt_scratch_ + tq::paged_prompt_scratch_bytes(dim, sms_));
        TQ_CUDA(cudaDeviceSynchronize());   // the first call may come on any stream
        h_status_ = tq::status_word_take(device_);
        d_status_ = static_cast<unsigned int*>(tq::pinned_host_device_alias(h_status_));
        TQ_REQUIRE(d_status_ != nullptr, "paged cache: the status word is not mapped for the device");
    }
    PagedKVCache(const PagedKVCache&) = delete;
    PagedKVCache& operator=(const PagedKVCache&) = delete;
    ~PagedKVCache() {
        int cur = -1;
        const bool other = cudaGetDevice(&cur) == cudaSuccess && cur != device_;
        if (other) cudaSetDevice(device_);
        if (!use_.only_legacy()) cudaDeviceSynchronize();   // (the buffers then find nothing pending)
        scratch_.release();
        state_.release();
        layers_.clear();
        if (h_status_) tq::status_word_return(h_status_, device_);
        if (other) cudaSetDevice(cur);
    }

    void plan(const int* rows, const int* counts, int n, int tokens, int max_count, int* starts, int* lengths, int* slots, int* positions, int* tables,
              int tables_width, cudaStream_t st) {
        TQ_REQUIRE(n >= 0 && n <= b_.max_requests, "paged plan: more requests than the cache was made for");
        TQ_REQUIRE(tokens >= 0 && tokens <= max_tokens_, "paged plan: more tokens than the cache was made for");
        TQ_REQUIRE(max_count >= 0, "paged plan: negative max_count");
        TQ_REQUIRE(n == 0 || counts, "paged plan: NULL counts");
        TQ_REQUIRE(!tables || tables_width > 0, "paged plan: tables without a width");
        for (const void* p : {static_cast<const void*>(starts), static_cast<const void*>(lengths), static_cast<const void*>(slots),
                              static_cast<const void*>(positions), static_cast<const void*>(tables)})
            TQ_REQUIRE(!p || tq::is_device_pointer(p), "paged plan: outputs must be device pointers");
        begin(st);
        tq::PagedPlanArgs a{b_, staged(rows, n, 0, st), staged(counts, n, b_.max_requests, st), n, tokens, max_count, starts, lengths, slots, positions, tables,
                            tables_width, d_status_, sms_};
        tq::launch_paged_plan(a, st);
        plan_ = {n, tokens, std::min(max_count, tokens)};
        tree_ = false;
    }
    void tree(const int* parents, int tokens, int* positions, cudaStream_t st) {
        TQ_REQUIRE(plan_.n >= 0, "paged tree: no plan in force");
        TQ_REQUIRE(tokens == plan_.tokens, "paged tree: the plan is for " + std::to_string(plan_.tokens) + " tokens");
        TQ_REQUIRE(!parents || tokens == 0 || tq::is_device_pointer(parents), "paged tree: parents must be a device pointer");
        TQ_REQUIRE(!positions || tokens == 0 || tq::is_device_pointer(positions), "paged tree: positions must be a device pointer");
        // (a request's CTA reads all of its parents before it writes its positions, but others' it does not know)
        TQ_REQUIRE(positions == parents || tq::ranges_apart(positions, 4ul * tokens, parents, 4ul * tokens),
                   "paged tree: positions must not be where the parents are, but for the same address");
        begin(st);
        tq::launch_paged_tree({b_, parents, positions, plan_, d_status_}, st);
        tree_ = true;
    }
    void keep(const int* path, int width, const int* kept, int n, int* lengths, cudaStream_t st) {
        TQ_REQUIRE(plan_.n >= 0, "paged keep: no plan in force");
        TQ_REQUIRE(n == plan_.n, "paged keep: the plan is for " + std::to_string(plan_.n) + " requests");
        TQ_REQUIRE(width > 0, "paged keep: a path has room for one token at least");
        if (n == 0) return;
        TQ_REQUIRE(tq::is_device_pointer(path) && tq::is_device_pointer(kept) && (!lengths || tq::is_device_pointer(lengths)),
                   "paged keep: paths, their lengths and results must be device pointers");
        // (the kernel behind the bookkeeping reads both again)
        TQ_REQUIRE(tq::ranges_apart(lengths, 4ul * n, kept, 4ul * n) && tq::ranges_apart(lengths, 4ul * n, path, 4ul * n * width),
                   "paged keep: lengths must not be where the paths or their lengths are");
        begin(st);
        tq::launch_paged_keep({b_, path, kept, lengths, n, width, heads_, static_cast<int>(layers_.size()), plan_, d_status_, sms_}, dim_, st);
        plan_.n = -1;
    }
    void truncate(const int* rows, const int* lengths, int n, cudaStream_t st) {
        TQ_REQUIRE(n >= 0 && n <= b_.max_requests, "paged truncate: more requests than the cache was made for");
        TQ_REQUIRE(n == 0 || lengths, "paged truncate: NULL lengths");
        if (n == 0) return;
        begin(st);
        tq::PagedPlanArgs a{};
        a.b = b_;
        a.rows = staged(rows, n, 0, st);
        a.counts = staged(lengths, n, b_.max_requests, st);
        a.n = n;
        a.status = d_status_;
        a.sms = sms_;
        tq::launch_paged_truncate(a, st);
        plan_.n = -1;
    }
    void append(int layer, const void* keys, const void* values, int dtype, int tokens, long key_stride, long value_stride, cudaStream_t st) {
        check_layer(layer);
        TQ_REQUIRE(plan_.n >= 0, "paged append: no plan in force");
        TQ_REQUIRE(dtype == TQ_F32 || dtype == TQ_F16, "paged append: keys and values must be fp32 or fp16");
        TQ_REQUIRE(tokens == plan_.tokens, "paged append: the plan is for " + std::to_string(plan_.tokens) + " tokens");
        if (plan_.n == 0 || plan_.most == 0) return;
        TQ_REQUIRE(tq::is_device_pointer(keys) && tq::is_device_pointer(values), "paged append: keys and values must be device pointers");
        const long row = static_cast<long>(heads_) * dim_;
        TQ_REQUIRE(key_stride >= row && value_stride >= row, "paged append: a token's stride is shorter than its heads");
        begin(st);
        tq::PagedAppendArgs a{b_.header, b_.pieces, layers_[static_cast<size_t>(layer)].as<uint8_t>(), keys, values, key_stride, value_stride, heads_,
                              b_.page_tokens, plan_, d_status_};
        tq::launch_paged_append(a, dim_, dtype == TQ_F16, st);
    }
    void read(int layer, const int* pages, int n, void* keys, void* values, int dtype, cudaStream_t st) {
        check_layer(layer);
        TQ_REQUIRE(dtype == TQ_F32 || dtype == TQ_F16, "paged read: keys and values must be fp32 or fp16");
        TQ_REQUIRE(n >= 0 && static_cast<long>(n) * heads_ < (1l << 31), "paged read: bad number of pages");
        if (n == 0 || (!keys && !values)) return;
        TQ_REQUIRE(tq::is_device_pointer(pages), "paged read: page numbers must be a device pointer");
        for (const void* p : {static_cast<const void*>(keys), static_cast<const void*>(values)}) {
            TQ_REQUIRE(!p || tq::is_device_pointer(p), "paged read: keys and values must be device pointers");
            TQ_REQUIRE(reinterpret_cast<uintptr_t>(p) % 16 == 0, "paged read: keys and values must be 16-byte aligned");
        }
        begin(st);
        tq::PagedReadArgs a{layers_[static_cast<size_t>(layer)].as<uint8_t>(), pages, keys, values, n, heads_, b_.page_tokens, b_.num_pages, d_status_};
        tq::launch_paged_read(a, dim_, dtype == TQ_F16, st);
    }
    void attention(int layer, const void* q, int tokens, int q_heads, long q_stride, int window, float scale, void* out, long out_stride, float* lse, bool tree, cudaStream_t st) {
        check_layer(layer);
        TQ_REQUIRE(plan_.n >= 0, "paged attention: no plan in force");
        TQ_REQUIRE(!tree || tree_, "paged tree attention: the plan in force has no trees");
        TQ_REQUIRE(tokens == plan_.tokens, "paged attention: the plan is for " + std::to_string(plan_.tokens) + " tokens");
        TQ_REQUIRE(q_heads > 0 && q_heads % heads_ == 0, "paged attention: query heads must be a multiple of KV heads");
        TQ_REQUIRE(q_heads / heads_ <= 1024, "paged attention: more than 1024 query heads to a KV head");
        TQ_REQUIRE(window >= 0, "paged attention: negative window");
        TQ_REQUIRE(std::isfinite(scale) && scale >= 0.f, "paged attention: the scale must be finite, and 0 (1 / sqrt(head_dim)) or positive");
        if (plan_.n == 0 || plan_.most == 0) return;
        TQ_REQUIRE(tq::is_device_pointer(q) && tq::is_device_pointer(out) && (!lse || tq::is_device_pointer(lse)),
                   "paged attention: queries and results must be device pointers");
        const long row = static_cast<long>(q_heads) * dim_;
        TQ_REQUIRE(q_stride >= row && out_stride >= row, "paged attention: a token's stride is shorter than its heads");
        // (in place the rows of a request and head are written by the CTA that has read them, or by the kernel behind; anywhere else over the queries they
        // may be another's that has not)
        const tq::ByteRows from{q, 2ul * row, tokens, 2ul * q_stride}, to{out, 2ul * row, tokens, 2ul * out_stride}, logs{lse, 4ul * tokens * q_heads, lse ? 1 : 0};
        TQ_REQUIRE((out == q && (tokens == 1 || out_stride == q_stride)) || tq::rows_apart(to, from),
                   "paged attention: results must be where the queries are, with the same stride, or not where they are");
        TQ_REQUIRE(tq::rows_apart(logs, from) && tq::rows_apart(logs, to), "paged attention: lse must not be where queries or results are");
        begin(st);
        tq::PagedAttnArgs a{};
        a.b = b_;
        a.layer = layers_[static_cast<size_t>(layer)].as<uint8_t>();
        a.q = static_cast<const __half*>(q);
        a.out = static_cast<__half*>(out);
        a.lse = lse;
        a.q_stride = q_stride;
        a.out_stride = out_stride;
        a.sizes = plan_;
        a.heads = heads_;
        a.group = q_heads / heads_;
        a.window = window;
        a.page_shift = b_.page_tokens == 16 ? 4 : b_.page_tokens == 32 ? 5 : b_.page_tokens == 64 ? 6 : 7;
        a.scale_log2 = static_cast<float>((scale > 0.f ? static_cast<double>(scale) : 1.0 / std::sqrt(static_cast<double>(dim_))) * 1.4426950408889634);
        a.status = d_status_;
        if (tree) {
            tq::launch_paged_tree_attention(a, dim_, static_cast<long>(plan_.most) * a.group, scratch_.as<char>() + prompt_scratch_, sms_, st);
            return;
        }
        // Up to kFewRows query rows of a request (new tokens times query heads to a KV head) go to the kernel for few rows.  Over 4096 tokens of 16
        // requests, there and in the kernel for many: 14 rows 30 and 49 us; in a form that took several times 16 rows of a request, 21 rows 48 and
        // 48, 35 rows 67 and 49; 20 rows over 32768 tokens of 4 requests 132 and 132. The device finds the requests of each kernel; a batch of one
        // has one.
        const long max_rows = static_cast<long>(plan_.most) * a.group;
        const bool many = max_rows > tq::kFewRows;
        a.few_rows = many && plan_.n == 1 ? 0 : tq::kFewRows;
        if (many) tq::launch_paged_prompt(a, dim_, max_rows, scratch_.as<char>() + prompt_scratch_, sms_, st);
        if (a.few_rows) tq::launch_paged_attention(a, dim_, static_cast<int>(std::min<long>(max_rows, tq::kFewRows)), scratch_.as<void>(), sms_, st);
    }
    void check_status() {
        const unsigned int code = *static_cast<volatile unsigned int*>(h_status_);
        if (code == tq::kPagedOk) return;
        *static_cast<volatile unsigned int*>(h_status_) = tq::kPagedOk;
        static const std::string what[] = {"", "a row outside the tables, or twice in a batch",
                                           "a negative count, one above max_count, or more tokens in all than announced",
                                           "a request would be longer than max_pages_per_request pages", "not enough free pages",
                                           "truncation to a length that the request does not have", "a page number outside the cache",
                                           "a wait on the device ran out",
                                           "the plan on the device is not the one that a call was made for",
                                           "parents that make no tree, or a tree of more than " + std::to_string(tq::kPagedTreeNodes) + " nodes",
                                           "a path that is not an ascending list of a request's new tokens"};
        throw tq::Error("paged cache: " + what[code < 11 ? code : 0]);
    }
    int free_pages() {
        tq::ensure_device(device_);
        TQ_CUDA(cudaDeviceSynchronize());
        int n = 0;
        TQ_CUDA(cudaMemcpy(&n, &b_.header->free_pages, 4, cudaMemcpyDeviceToHost));
        return n;
    }

private:
    void check_layer(int layer) const { TQ_REQUIRE(layer >= 0 && layer < static_cast<int>(layers_.size()), "Layer index out of range"); }
    void begin(cudaStream_t st) {
        tq::ensure_device(device_);
        use_.note(st);
    }
    // Host numbers on the device.  They are the caller's again when the call returns: a copy from pageable memory is staged before it returns, one from
    // page-locked memory reads it when the stream comes to it, so that the caller's numbers go through pageable memory first, whatever they are in.
    const int* staged(const int* p, int n, int at, cudaStream_t st) {
        if (!p || n == 0 || tq::is_device_pointer(p)) return p;
        TQ_REQUIRE(!tq::stream_is_capturing(st), "paged cache: a captured plan needs its numbers in device memory");
        std::copy(p, p + n, numbers_.begin());
        TQ_CUDA(cudaMemcpyAsync(staged_ + at, numbers_.data(), 4ul * n, cudaMemcpyHostToDevice, st));
        return staged_ + at;
    }

    int heads_, dim_, max_tokens_, device_ = 0, sms_ = 0;
    tq::PagedSizes plan_{-1, 0, 0};   // of the plan in force (n < 0: none)
    bool tree_ = false;               // its tokens are trees
    size_t prompt_scratch_ = 0;
    tq::StreamUse use_;
    std::vector<DeviceBuffer> layers_;
    DeviceBuffer state_, scratch_;
    int* staged_ = nullptr;
    std::vector<int> numbers_;
    tq::PagedBatch b_{};
    unsigned int* h_status_ = nullptr;
    unsigned int* d_status_ = nullptr;
};

}  // namespace turboquant

struct tq_paged_cache_s {
    std::unique_ptr<turboquant::PagedKVCache> cache;
};

using namespace tq;

namespace {
turboquant::PagedKVCache* paged(tq_paged_cache_t c) {
    TQ_REQUIRE(c && c->cache, "paged cache: NULL handle");
    return c->cache.get();
}
cudaStream_t cuda_stream(void* s) { return static_cast<cudaStream_t>(s); }
}  // namespace

extern "C" {

tq_paged_cache_t tq_paged_cache_create(int num_layers, int num_heads, int head_dim, int num_pages, int page_tokens, int max_requests,
                                       int max_pages_per_request, int max_tokens) {
    return guarded<tq_paged_cache_t>(nullptr, nullptr, [&]() -> tq_paged_cache_t {
        auto c = std::make_unique<turboquant::PagedKVCache>(num_layers, num_heads, head_dim, num_pages, page_tokens, max_requests, max_pages_per_request, max_tokens);
        return new tq_paged_cache_s{std::move(c)};
    });
}
void tq_paged_cache_free(tq_paged_cache_t cache) { delete cache; }

int tq_paged_plan(tq_paged_cache_t cache, const int* rows, const int* counts, int n, int tokens, int max_count, int* starts, int* lengths, int* slots,
                  int* positions, int* tables, int tables_width, void* stream) {
    return guarded<int>(0, -1, [&]() {
        paged(cache)->plan(rows, counts, n, tokens, max_count, starts, lengths, slots, positions, tables, tables_width, cuda_stream(stream));
        return 0;
    });
}
int tq_paged_truncate(tq_paged_cache_t cache, const int* rows, const int* lengths, int n, void* stream) {
    return guarded<int>(0, -1, [&]() {
        paged(cache)->truncate(rows, lengths, n, cuda_stream(stream));
        return 0;
    });
}
int tq_paged_tree(tq_paged_cache_t cache, const int* parents, int tokens, int* positions, void* stream) {
    return guarded<int>(0, -1, [&]() {
        paged(cache)->tree(parents, tokens, positions, cuda_stream(stream));
        return 0;
    });
}
int tq_paged_keep(tq_paged_cache_t cache, const int* path, int width, const int* kept, int n, int* lengths, void* stream) {
    return guarded<int>(0, -1, [&]() {
        paged(cache)->keep(path, width, kept, n, lengths, cuda_stream(stream));
        return 0;
    });
}
int tq_paged_append(tq_paged_cache_t cache, int layer, const void* keys, const void* values, int dtype, int tokens, long key_stride, long value_stride,
                    void* stream) {
    return guarded<int>(0, -1, [&]() {
        paged(cache)->append(layer, keys, values, dtype, tokens, key_stride, value_stride, cuda_stream(stream));
        return 0;
    });
}
int tq_paged_read(tq_paged_cache_t cache, int layer, const int* pages, int n, void* keys, void* values, int dtype, void* stream) {
    return guarded<int>(0, -1, [&]() {
        paged(cache)->read(layer, pages, n, keys, values, dtype, cuda_stream(stream));
        return 0;
    });
}
int tq_paged_attention(tq_paged_cache_t cache, int layer, const void* queries_fp16, int tokens, int q_heads, long q_stride, int window, float scale,
                       void* out_fp16, long out_stride, float* lse, void* stream) {
    return guarded<int>(0, -1, [&]() {
        paged(cache)->attention(layer, queries_fp16, tokens, q_heads, q_stride, window, scale, out_fp16, out_stride, lse, false, cuda_stream(stream));
        return 0;
    });
}
int tq_paged_tree_attention(tq_paged_cache_t cache, int layer, const void* queries_fp16, int tokens, int q_heads, long q_stride, int window, float scale,
                            void* out_fp16, long out_stride, float* lse, void* stream) {
    return guarded<int>(0, -1, [&]() {
        paged(cache)->attention(layer, queries_fp16, tokens, q_heads, q_stride, window, scale, out_fp16, out_stride, lse, true, cuda_stream(stream));
        return 0;
    });
}
int tq_paged_status(tq_paged_cache_t cache) {
    return guarded<int>(0, -1, [&]() {
        paged(cache)->check_status();
        return 0;
    });
}
int tq_paged_free_pages(tq_paged_cache_t cache) {
    return guarded<int>(0, -1, [&]() { return paged(cache)->free_pages(); });
}

}  // extern "C"
