// Rows of a paged cache: the store of a batch's new tokens (g4_paged_append)
// and the accepted drafts' rows moved together (g4_paged_commit).
#include "paged.h"
#include "ref_math.h"

namespace g4 {

// ---- append -----------------------------------------------------------------
//
// Per token: q' = rope(q wq / rms(q)), k' = rope(k wk / rms(k)), v' = v / rms(v),
// rms(x) = sqrt(mean x^2 + eps), by wave_norm_rope: the values every other prep of
// this library stores, before the rounding to the cache's type. One workgroup a
// token: its threads evaluate the cos and sin of the token's angles (in f64, as
// the other preps do), its four waves take the head slots (q heads, k heads, v
// heads) in turn. A wave requests its first row before it looks for the token's
// sequence, page and position, which are three dependent loads. Bound by its
// bytes (four prompts of 1000 tokens, e4m3, head_dim 512: 21 us at the rate of
// a large copy), and for few tokens by those loads: 512 tokens take 5.1 us.
struct AppendArgs {
    const float* __restrict__ q;
    const float* __restrict__ k;
    const float* __restrict__ v;
    const uint16_t* __restrict__ q_weight;
    const uint16_t* __restrict__ k_weight;
    const float* __restrict__ inv;
    uint16_t* __restrict__ q_out;
    void* __restrict__ k_pool;
    void* __restrict__ v_pool;
    uint64_t q_stride, k_stride, v_stride;
    uint32_t nqh, nkh;  // 0: no q / no k and v
    float eps;
    PagedBatchDev b;
};

// f32 -> e4m3, nearest even, values past 448 to 448 (the conversion alone makes them NaN).
__device__ __forceinline__ uint8_t f2e4m3(float x) {
    const float y = x != x ? x : fminf(fmaxf(x, -448.0f), 448.0f);
    return (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false) & 0xff);
}

// The sequence of token t: the last one that starts at or before it. 64 starts
// a step, one a lane.
__device__ __forceinline__ unsigned paged_find_seq(const PagedBatchDev& b, unsigned t, unsigned lane) {
    unsigned count = 0;
    for (unsigned s0 = 0; s0 < b.n_seqs; s0 += 64) {
        const unsigned s = s0 + lane;
        count += __popcll(__ballot(s < b.n_seqs && b.start[s] <= (int32_t)t));
    }
    return count;  // one past the sequence
}

template <int HD, bool F8>
__global__ __launch_bounds__(kWG) void k_paged_append(const AppendArgs a) {
    constexpr int J = HD / 64, PJ = J / 2;
    constexpr unsigned NP = HD / 2;
    __shared__ float rc[NP], rs[NP];
    const unsigned t = blockIdx.x, lane = threadIdx.x & 63;
    const unsigned wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned S = a.nqh + 2 * a.nkh;
    auto row_src = [&](unsigned slot) __attribute__((always_inline)) {
        const unsigned r = slot - a.nqh;
        return slot < a.nqh ? a.q + t * a.q_stride + (uint64_t)slot * HD
                            : (r < a.nkh ? a.k + t * a.k_stride + (uint64_t)r * HD
                                         : a.v + t * a.v_stride + (uint64_t)(r - a.nkh) * HD);
    };
    float x[J];
    unsigned slot = wave;
    if (slot < S) {
        const float* src = row_src(slot);
#pragma unroll
        for (int j = 0; j < J; j++) x[j] = src[lane + 64 * j];
    }
    const unsigned found = paged_find_seq(a.b, t, lane);
    if (found == 0) return;  // uniform: padding before the first sequence
    const unsigned s = found - 1;
    const PagedSeq sq = paged_seq(a.b, s);
    if (t < sq.start || t - sq.start >= sq.n) return;  // uniform: padding behind a sequence
    const unsigned row = sq.ctx + (t - sq.start);
    const unsigned pos = a.b.positions ? (unsigned)max(a.b.positions[t], 0) : row;
    if (threadIdx.x < NP) {
        const float ang = (float)pos * a.inv[threadIdx.x];  // rope_angle's expression
        f64_cos_sin(ang, rc[threadIdx.x], rs[threadIdx.x]);
    }
    const unsigned page = row < paged_rows(a.b)
                              ? (unsigned)a.b.table[(uint64_t)s * a.b.table_stride + (row >> a.b.page_shift)]
                              : 0xffffffffu;
    const uint64_t cache_row = ((uint64_t)page << a.b.page_shift) + (row & ((1u << a.b.page_shift) - 1u));
    uint32_t wq[J], wk[J];
#pragma unroll
    for (int j = 0; j < J; j++) {
        wq[j] = a.nqh ? a.q_weight[lane + 64 * j] : 0u;
        wk[j] = a.nkh ? a.k_weight[lane + 64 * j] : 0u;
    }
    __syncthreads();
    RopeLane<PJ> rl;
#pragma unroll
    for (int p = 0; p < PJ; p++) {
        rl.c[p] = rc[lane + 64 * p];
        rl.s[p] = rs[lane + 64 * p];
    }
    while (slot < S) {  // uniform per wave
        const unsigned next = slot + kWG / 64;
        float xn[J];
        {  // the next row's request (the last slot re-reads its own) before this one's stores
            const float* src = row_src(next < S ? next : slot);
#pragma unroll
            for (int j = 0; j < J; j++) xn[j] = src[lane + 64 * j];
        }
        const bool is_q = slot < a.nqh, is_k = !is_q && slot < a.nqh + a.nkh, rope = is_q || is_k;
        uint32_t wb[J];
#pragma unroll
        for (int j = 0; j < J; j++) wb[j] = is_q ? wq[j] : wk[j];
        wave_norm_rope<J>(x, wb, rope, rope, rl, a.eps);
        if (is_q) {
            uint16_t* dst = a.q_out + ((uint64_t)t * a.nqh + slot) * HD;
#pragma unroll
            for (int j = 0; j < J; j++) dst[lane + 64 * j] = f2h(x[j]);
        } else if (page < a.b.num_pages) {
            const unsigned h = is_k ? slot - a.nqh : slot - a.nqh - a.nkh;
            const uint64_t at = (cache_row * a.nkh + h) * HD + lane;
            if constexpr (F8) {
                uint8_t* dst = static_cast<uint8_t*>(is_k ? a.k_pool : a.v_pool) + at;
#pragma unroll
                for (int j = 0; j < J; j++) dst[64 * j] = f2e4m3(x[j]);
            } else {
                uint16_t* dst = static_cast<uint16_t*>(is_k ? a.k_pool : a.v_pool) + at;
#pragma unroll
                for (int j = 0; j < J; j++) dst[64 * j] = f2h(x[j]);
            }
        }
        slot = next;
#pragma unroll
        for (int j = 0; j < J; j++) x[j] = xn[j];
    }
}

// ---- commit -----------------------------------------------------------------
//
// One thread a (sequence, 16-byte column of a row) of a pool. It reads a batch of
// the path's rows before it writes any. That is enough: the path ascends, so
// path[d] >= d, and a row written at step d is no later step's source (those
// are above path[d]); other columns belong to other threads. Bound by its
// dependent loads (lengths, path, page, row: 5 us for one sequence in 15 layers,
// 8 for 64 in 10), which a batch of eight rows has side by side.
struct CommitPool {
    void* p;
    uint32_t row_bytes;
    uint32_t pieces;  // row_bytes / 16
};
struct CommitArgs {
    CommitPool pool[2 * G4_COMMIT_MAX_CACHES];
    const int32_t* __restrict__ path;
    const int32_t* __restrict__ accepted;
    int32_t* __restrict__ new_ctx;
    uint32_t path_stride;
    PagedBatchDev b;
};

constexpr int kCommitBatch = 8;

__global__ __launch_bounds__(kWG) void k_paged_commit(const CommitArgs a) {
    const CommitPool pool = a.pool[blockIdx.y];
    const unsigned i = blockIdx.x * kWG + threadIdx.x;  // below 2^31 (checked on the host)
    const unsigned s = i / pool.pieces, piece = i % pool.pieces;
    if (s >= a.b.n_seqs) return;
    const PagedSeq sq = paged_seq(a.b, s);
    const unsigned n = min((unsigned)max(a.accepted[s], 0), a.path_stride);
    const int32_t* path = a.path + (uint64_t)s * a.path_stride;
    const int32_t* table = a.b.table + (uint64_t)s * a.b.table_stride;
    char* base = static_cast<char*>(pool.p) + (uint64_t)piece * 16;
    auto place = [&](unsigned row) __attribute__((always_inline)) -> char* {  // nullptr: no page
        if (row >= paged_rows(a.b)) return nullptr;
        const unsigned page = (unsigned)table[row >> a.b.page_shift];
        if (page >= a.b.num_pages) return nullptr;
        return base + (((uint64_t)page << a.b.page_shift) + (row & ((1u << a.b.page_shift) - 1u))) * pool.row_bytes;
    };
    int prev = -1;
    unsigned len = 0;
    bool more = true;
    for (unsigned d0 = 0; more && d0 < n; d0 += kCommitBatch) {
        u32x4 v[kCommitBatch];
        bool have[kCommitBatch];
#pragma unroll
        for (int u = 0; u < kCommitBatch; u++) {
            const unsigned d = d0 + u;
            const int at = d < n ? path[d] : -1;
            more = more && at > prev && (unsigned)at < sq.n;
            prev = at;
            const char* src = more ? place(sq.ctx + (unsigned)at) : nullptr;
            have[u] = src != nullptr;
            if (have[u]) v[u] = ldg<u32x4>(src);
            len += more;
        }
#pragma unroll
        for (int u = 0; u < kCommitBatch; u++) {
            char* dst = have[u] ? place(sq.ctx + d0 + u) : nullptr;
            if (dst) stg<u32x4>(dst, v[u]);
        }
    }
    if (blockIdx.y == 0 && piece == 0) a.new_ctx[s] = (int32_t)(sq.ctx + len);
}

int paged_check(const char* who, const g4_paged_cache* c, const g4_paged_batch* b, PagedBatchDev* out) {
    if (!c || !b) return fail(G4_EINVAL, "%s: NULL cache or batch", who);
    if (c->head_dim != 256 && c->head_dim != 512)
        return fail(G4_EINVAL, "%s: head_dim %u unsupported (256 or 512)", who, c->head_dim);
    if (c->page_size < 16 || c->page_size > 1024 || (c->page_size & (c->page_size - 1)))
        return fail(G4_EINVAL, "%s: page_size %u is not a power of two in [16, 1024]", who, c->page_size);
    if (c->dtype != G4_KV_F16 && c->dtype != G4_KV_E4M3) return fail(G4_EINVAL, "%s: cache dtype %u", who, c->dtype);
    if (c->num_kv_heads == 0 || c->num_kv_heads > 1024)
        return fail(G4_EINVAL, "%s: num_kv_heads %u (1 to 1024)", who, c->num_kv_heads);
    if (c->num_pages == 0 || c->num_pages > 0x7fffffffu) return fail(G4_EINVAL, "%s: num_pages %u", who, c->num_pages);
    if (c->reserved || b->reserved) return fail(G4_EINVAL, "%s: reserved fields must be 0", who);
    if (!c->k_pool || !c->v_pool) return fail(G4_EINVAL, "%s: NULL pool", who);
    if ((reinterpret_cast<uintptr_t>(c->k_pool) | reinterpret_cast<uintptr_t>(c->v_pool)) & 15)
        return fail(G4_EINVAL, "%s: pools must be 16-byte aligned", who);
    if (!b->block_table || !b->token_start || !b->ctx_lens)
        return fail(G4_EINVAL, "%s: NULL block_table, token_start or ctx_lens", who);
    if (b->n_seqs == 0 || b->n_seqs > 65535) return fail(G4_EINVAL, "%s: %u sequences (1 to 65535)", who, b->n_seqs);
    if (b->table_stride == 0 || (uint64_t)b->table_stride * c->page_size > (1ull << 30))
        return fail(G4_EINVAL, "%s: table_stride %u of %u-row pages (1 to 2^30 rows)", who, b->table_stride, c->page_size);
    if (b->n_tokens > (1u << 22)) return fail(G4_EINVAL, "%s: %u tokens (at most 2^22)", who, b->n_tokens);
    if (b->n_tokens && b->max_tokens == 0) return fail(G4_EINVAL, "%s: max_tokens 0", who);
    const uint32_t max_tokens = b->max_tokens < b->n_tokens ? b->max_tokens : b->n_tokens;
    if (b->tree_mask && (uint64_t)b->mask_words * 64 < max_tokens)
        return fail(G4_EINVAL, "%s: %u mask words for %u tokens a sequence", who, b->mask_words, max_tokens);
    out->table = b->block_table;
    out->start = b->token_start;
    out->ctx = b->ctx_lens;
    out->positions = b->positions;
    out->mask = b->tree_mask;
    out->n_seqs = b->n_seqs;
    out->table_stride = b->table_stride;
    out->n_tokens = b->n_tokens;
    out->max_tokens = max_tokens;
    out->mask_words = b->mask_words;
    out->page_shift = (uint32_t)__builtin_ctz(c->page_size);
    out->num_pages = c->num_pages;
    return G4_OK;
}

}  // namespace g4

using namespace g4;

namespace {

// Whether two arrays of 4-byte elements share one.
bool overlap(const int32_t* x, uint64_t nx, const int32_t* y, uint64_t ny) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(x), b = reinterpret_cast<uintptr_t>(y);
    return a < b + ny * 4 && b < a + nx * 4;
}
// Whether two of n pools are one, by open addressing over twice as many places as there may be pools.
bool repeated(const CommitPool* pool, uint32_t n) {
    constexpr uint32_t PLACES = 4 * G4_COMMIT_MAX_CACHES;
    const void* seen[PLACES] = {};
    for (uint32_t i = 0; i < n; i++) {
        uint32_t at = (uint32_t)((reinterpret_cast<uintptr_t>(pool[i].p) >> 4) * 0x9E3779B97F4A7C15ull >> 56);
        static_assert(PLACES == 256, "the hash's top byte");
        for (; seen[at]; at = (at + 1) % PLACES)
            if (seen[at] == pool[i].p) return true;
        seen[at] = pool[i].p;
    }
    return false;
}

// The pools go by value in the kernel arguments.
int commit(const g4_paged_cache* caches, uint32_t n_caches, const g4_paged_batch* batch, const int32_t* path,
           uint32_t path_stride, const int32_t* n_accepted, int32_t* new_ctx_lens, void* stream) {
    CommitArgs a;
    uint32_t most = 0;
    for (uint32_t i = 0; i < n_caches; i++) {
        const g4_paged_cache& c = caches[i];
        g4_paged_batch plain = batch ? *batch : g4_paged_batch{};
        plain.positions = nullptr;
        plain.tree_mask = nullptr;
        const int rc = paged_check("pagedCommit", &c, batch ? &plain : nullptr, &a.b);
        if (rc) return rc;
        if (c.page_size != caches[0].page_size || c.num_pages != caches[0].num_pages)
            return fail(G4_EINVAL, "pagedCommit: cache %u has %u pages of %u rows, cache 0 %u of %u", i, c.num_pages,
                        c.page_size, caches[0].num_pages, caches[0].page_size);
        const uint32_t row_bytes = c.num_kv_heads * c.head_dim * (c.dtype == G4_KV_E4M3 ? 1u : 2u);
        a.pool[2 * i] = {c.k_pool, row_bytes, row_bytes / 16};
        a.pool[2 * i + 1] = {c.v_pool, row_bytes, row_bytes / 16};
        if (row_bytes / 16 > most) most = row_bytes / 16;
    }
    if (new_ctx_lens == batch->ctx_lens) return fail(G4_EINVAL, "pagedCommit: new_ctx_lens is ctx_lens itself");
    // Written while other workgroups still read these.
    const uint64_t seqs = batch->n_seqs;
    if (overlap(new_ctx_lens, seqs, batch->ctx_lens, seqs) || overlap(new_ctx_lens, seqs, n_accepted, seqs) ||
        overlap(new_ctx_lens, seqs, path, seqs * path_stride) || overlap(new_ctx_lens, seqs, batch->token_start, seqs + 1) ||
        overlap(new_ctx_lens, seqs, batch->block_table, seqs * batch->table_stride))
        return fail(G4_EINVAL, "pagedCommit: new_ctx_lens lies over ctx_lens, token_start, block_table, n_accepted or path");
    if (repeated(a.pool, 2 * n_caches)) return fail(G4_EINVAL, "pagedCommit: a pool is named twice (its rows would move twice)");
    a.path = path;
    a.accepted = n_accepted;
    a.new_ctx = new_ctx_lens;
    a.path_stride = path_stride;
    const uint64_t threads = (uint64_t)batch->n_seqs * most;
    if (threads > 0x7fffff00u) return fail(G4_EINVAL, "pagedCommit: %u sequences of %u-byte rows are too many", batch->n_seqs, most * 16);
    G4_LAUNCH(k_paged_commit, dim3((uint32_t)((threads + kWG - 1) / kWG), 2 * n_caches), dim3(kWG), 0, as_stream(stream), a);
    G4_CHECK_LAUNCH("pagedCommit");
    return G4_OK;
}

}  // namespace

extern "C" {

int g4_paged_append(const g4_paged_cache* cache, const g4_paged_batch* batch, const float* q, const float* k,
                    const float* v, const uint16_t* q_weight, const uint16_t* k_weight, const float* rope_inv_freq,
                    uint16_t* q_out, const g4_paged_append_params* p, void* stream) {
    AppendArgs a = {};
    const int rc = paged_check("pagedAppend", cache, batch, &a.b);
    if (rc) return rc;
    if (!p || !rope_inv_freq) return fail(G4_EINVAL, "pagedAppend: NULL params or rope_inv_freq");
    const bool has_q = q || q_weight || q_out, has_kv = k || v || k_weight;
    if (has_q && (!q || !q_weight || !q_out)) return fail(G4_EINVAL, "pagedAppend: q, q_weight and q_out go together");
    if (has_kv && (!k || !v || !k_weight)) return fail(G4_EINVAL, "pagedAppend: k, v and k_weight go together");
    if (!has_q && !has_kv) return fail(G4_EINVAL, "pagedAppend: neither q nor k and v");
    const uint64_t hd = cache->head_dim, nq = (uint64_t)p->num_q_heads * hd, nk = (uint64_t)cache->num_kv_heads * hd;
    if (has_q && (p->num_q_heads == 0 || p->num_q_heads > 8192))
        return fail(G4_EINVAL, "pagedAppend: num_q_heads %u (1 to 8192)", p->num_q_heads);
    if (!(p->eps >= 0.0f)) return fail(G4_EINVAL, "pagedAppend: eps %g", (double)p->eps);
    a.q_stride = p->q_stride ? p->q_stride : nq;
    a.k_stride = p->k_stride ? p->k_stride : nk;
    a.v_stride = p->v_stride ? p->v_stride : nk;
    if ((has_q && a.q_stride < nq) || (has_kv && (a.k_stride < nk || a.v_stride < nk)))
        return fail(G4_EINVAL, "pagedAppend: a token stride shorter than the token's heads");
    if ((a.q_stride | a.k_stride | a.v_stride) > (1ull << 32)) return fail(G4_EINVAL, "pagedAppend: token stride too long");
    if (((a.q_stride | a.k_stride | a.v_stride) & 3) ||
        ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
          reinterpret_cast<uintptr_t>(q_out)) & 15))
        return fail(G4_EINVAL, "pagedAppend: rows must be 16-byte aligned");
    if (batch->n_tokens == 0) return G4_OK;
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_weight = q_weight;
    a.k_weight = k_weight;
    a.inv = rope_inv_freq;
    a.q_out = q_out;
    a.k_pool = cache->k_pool;
    a.v_pool = cache->v_pool;
    a.nqh = has_q ? p->num_q_heads : 0;
    a.nkh = has_kv ? cache->num_kv_heads : 0;
    a.eps = p->eps;
    const dim3 grid(batch->n_tokens), block(kWG);
    hipStream_t st = as_stream(stream);
    const bool f8 = cache->dtype == G4_KV_E4M3;
    if (cache->head_dim == 512) {
        if (f8) G4_LAUNCH((k_paged_append<512, true>), grid, block, 0, st, a);
        else G4_LAUNCH((k_paged_append<512, false>), grid, block, 0, st, a);
    } else {
        if (f8) G4_LAUNCH((k_paged_append<256, true>), grid, block, 0, st, a);
        else G4_LAUNCH((k_paged_append<256, false>), grid, block, 0, st, a);
    }
    G4_CHECK_LAUNCH("pagedAppend");
    return G4_OK;
}

int g4_paged_commit(const g4_paged_cache* caches, uint32_t n_caches, const g4_paged_batch* batch, const int32_t* path,
                    uint32_t path_stride, const int32_t* n_accepted, int32_t* new_ctx_lens, void* stream) {
    if (!caches || n_caches == 0 || n_caches > G4_COMMIT_MAX_CACHES)
        return fail(G4_EINVAL, "pagedCommit: %u caches (1 to %d)", n_caches, G4_COMMIT_MAX_CACHES);
    if (!path || !n_accepted || !new_ctx_lens) return fail(G4_EINVAL, "pagedCommit: NULL path, n_accepted or new_ctx_lens");
    if (path_stride == 0 || path_stride > (1u << 30)) return fail(G4_EINVAL, "pagedCommit: path_stride %u", path_stride);
    return commit(caches, n_caches, batch, path, path_stride, n_accepted, new_ctx_lens, stream);
}

}  // extern "C"
