// The paged cache and the batch over it, as the kernels see them (paged_attn.hip,
// paged_store.hip).
//
// What a batch's device arrays hold is not known on the host, so every value
// read from them is brought into range here before it is used: token ranges
// into [0, n_tokens) and at most max_tokens long, committed rows into the block
// table's rows, page ids checked against the pool (a row without a page is
// neither written nor attended). No content of them leads to an access outside
// the buffers.
#pragma once

#include "common.h"
#include "tables.h"

namespace g4 {

struct PagedBatchDev {
    const int32_t* __restrict__ table;      // [n_seqs][table_stride]
    const int32_t* __restrict__ start;      // [n_seqs + 1]
    const int32_t* __restrict__ ctx;        // [n_seqs]
    const int32_t* __restrict__ positions;  // [n_tokens] or nullptr
    const uint64_t* __restrict__ mask;      // [n_tokens][mask_words] or nullptr
    uint32_t n_seqs;
    uint32_t table_stride;
    uint32_t n_tokens;
    uint32_t max_tokens;
    uint32_t mask_words;
    uint32_t page_shift;
    uint32_t num_pages;
};

// A sequence's tokens [start, start + n) and committed rows [0, ctx).
struct PagedSeq {
    unsigned start, n, ctx;
};

__device__ __forceinline__ unsigned paged_rows(const PagedBatchDev& b) { return b.table_stride << b.page_shift; }

__device__ __forceinline__ PagedSeq paged_seq_of(const PagedBatchDev& b, int32_t first, int32_t next, int32_t ctx) {
    const unsigned lo = min((unsigned)max(first, 0), b.n_tokens);
    const unsigned hi = min((unsigned)max(next, 0), b.n_tokens);
    PagedSeq q;
    q.start = lo;
    q.n = min(hi > lo ? hi - lo : 0u, b.max_tokens);
    q.ctx = min((unsigned)max(ctx, 0), paged_rows(b));
    return q;
}

__device__ __forceinline__ PagedSeq paged_seq(const PagedBatchDev& b, unsigned s) {
    return paged_seq_of(b, b.start[s], b.start[s + 1], b.ctx[s]);
}

// tanh(x) for |x| <= 1/2, to two half-steps of f32: x P(x^2), P the polynomial of degree 4 whose largest relative
// error on [0, 1/4] is least (Remez exchange: 2^-26.2).
__device__ __forceinline__ float tanh_near(float x) {
    const float z = x * x;
    float p = 0x1.18bd6ep-6f;
    p = __builtin_fmaf(p, z, -0x1.b20fdap-5f);
    p = __builtin_fmaf(p, z, 0x1.10e438p-3f);
    p = __builtin_fmaf(p, z, -0x1.5554a4p-2f);
    return x * __builtin_fmaf(p, z, 1.0f);
}
// And for every x, to three: above 1/2 as (1 - t) / (1 + t) with t = e^-2|x|, which cancels nothing there, its
// quotient rounded by one Newton step.
__device__ __forceinline__ float tanh_f32(float x) {
    const float t = __builtin_amdgcn_exp2f(-2.0f * kLog2e * fabsf(x));
    const float num = 1.0f - t, den = 1.0f + t;
    const float y = __builtin_amdgcn_rcpf(den), q = num * y;
    const float far = copysignf(__builtin_fmaf(__builtin_fmaf(-q, den, num), y, q), x);
    return fabsf(x) < 0.5f ? tanh_near(x) : far;
}

// Checks a batch and a cache on the host and fills the device form.
int paged_check(const char* who, const g4_paged_cache* c, const g4_paged_batch* b, PagedBatchDev* out);

}  // namespace g4
