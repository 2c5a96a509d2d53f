// Verification of drafted tokens (tq_drafts.cu): what its launch needs.
#pragma once

#include <cstdint>

#include "tq_common.cuh"

namespace tq {

constexpr int kDraftNodes = 1024;         // nodes of a request that are looked at
constexpr int kDraftVocab = 1 << 20;

struct VerifyArgs {
    const int* starts;     // [n + 1]
    const int* parents;    // [rows]
    const int* tokens;     // [rows]
    const void* target;    // [rows, vocab]
    const void* draft;     // or null: a point mass on each child's token
    const float* uniforms; // [rows]
    long target_stride, draft_stride;   // elements from row to row
    int rows, vocab, width;
    int segment;           // elements of a warp's part of a row
    int* path;             // [n, width]
    int* kept;             // [n]
    int* next;             // [n]
};
void launch_verify_drafts(VerifyArgs a, int n, bool half, cudaStream_t st);

}  // namespace tq
