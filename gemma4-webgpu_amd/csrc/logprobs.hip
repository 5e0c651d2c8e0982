// Log probabilities of given tokens, entropy and the best alternatives of rows
// of logits (g4_token_logprobs): what a step that verifies drafted tokens needs
// of them, next to the greedy head's argmax (lmhead.hip).
//
// z = cap tanh(x / cap) / T (or x / T), m = max z, S = sum e^(z - m),
// U = sum (z - m) e^(z - m):  log p(i) = z_i - m - log S,  entropy = log S - U / S.
// Bound by the logits' bytes, read once: a workgroup takes kLpChunk consecutive
// logits of a row into registers, so the maximum, the sums and the selection all
// work on what one pass has loaded. z is monotone in x, so maxima and ranks are
// taken on x itself and each element's z is evaluated once.
//
// Selection: candidates are 64-bit keys (order-preserving logit in the high half,
// inverted index in the low half), all different, so equal logits rank by index.
// The k-th largest of 64 groups' maxima bounds the k-th largest key from below;
// the few keys at or above it are collected in LDS and ranked by counting. Where
// that bound lets too many through (logits in ascending order, or most of them
// -inf), k rounds of a maximum below the last one take their place.
//
// Rows longer than a chunk leave (m, S, U) and k keys per chunk in the workspace;
// a second launch, a workgroup a row, joins them in a fixed order.
#include "paged.h"

namespace g4 {

constexpr unsigned kLpThreads = 256;
constexpr unsigned kLpElems = 32;  // logits a thread holds
constexpr unsigned kLpChunk = kLpThreads * kLpElems;
constexpr unsigned kLpMaxK = G4_LOGPROBS_MAX_TOP;
constexpr unsigned kLpGroups = 64;  // at least kLpMaxK
constexpr unsigned kLpCandidates = 1024;
static_assert(kLpGroups >= kLpMaxK, "the k-th largest group maximum must exist");

struct LogprobsArgs {
    const void* __restrict__ logits;
    const int32_t* __restrict__ tokens;
    float* __restrict__ logprobs;
    float* __restrict__ entropy;
    int32_t* __restrict__ top_ids;
    float* __restrict__ top_logprobs;
    float* __restrict__ part;      // [rows][chunks][4]: m (in z), S, U
    uint64_t* __restrict__ cand;   // [rows][chunks][k]
    uint64_t row_stride;
    uint32_t vocab, chunks, k;
    float cap, inv_cap, temperature, inv_temperature;
};

template <int DT>
struct LogitType {
    typedef uint16_t T;
};
template <>
struct LogitType<G4_LOGITS_F32> {
    typedef float T;
};

template <int DT>
__device__ __forceinline__ float logit_f32(typename LogitType<DT>::T v) {
    if constexpr (DT == G4_LOGITS_F32) return v;
    else if constexpr (DT == G4_LOGITS_F16) return h2f(v);
    else return __uint_as_float((uint32_t)v << 16);
}

// tanh(x) to f32 accuracy: below 1/2 the convergent of Lambert's continued
// fraction x / (1 + x^2 / (3 + x^2 / (5 + ...))) (its relative error there is under
// 2^-26), above it (1 - t) / (1 + t), t = e^(-2|x|), which loses no more than a bit.
__device__ __forceinline__ float tanh_f32(float x) {
    const float ax = fabsf(x), z = x * x;
    const float t = __builtin_amdgcn_exp2f(-2.0f * kLog2e * ax);
    const bool small = ax < 0.5f;
    const float num = small ? ax * (945.0f + z * (105.0f + z)) : 1.0f - t;
    const float den = small ? 945.0f + z * (420.0f + 15.0f * z) : 1.0f + t;
    const float y = __builtin_amdgcn_rcpf(den), q = num * y;
    return copysignf(__builtin_fmaf(__builtin_fmaf(-q, den, num), y, q), x);
}

// e^t for t <= 0 (0 from -200 on): the product's rounding error goes into the result.
__device__ __forceinline__ float exp_f32(float t) {
    constexpr float kLo = 1.92596299e-8f;  // log2(e) - kLog2e
    t = t < -200.0f ? -200.0f : t;         // -inf has no residual; a NaN stays one
    const float h = t * kLog2e;
    const float l = __builtin_fmaf(t, kLog2e, -h) + t * kLo;
    const float e = __builtin_amdgcn_exp2f(h);
    return __builtin_fmaf(e, l * 0.6931471805599453f, e);
}

__device__ __forceinline__ float logit_z(float x, const LogprobsArgs& a) {
    float z = x;
    if (a.cap > 0.0f && fabsf(x) != INFINITY) z = a.cap * tanh_f32(x * a.inv_cap);  // a mask of -inf stays one
    if (a.temperature != 1.0f) {
        const float q = z * a.inv_temperature;  // z / T with the quotient's residual
        const float r = __builtin_fmaf(-q, a.temperature, z);
        z = fabsf(z) == INFINITY ? z : __builtin_fmaf(r, a.inv_temperature, q);
    }
    return z;
}

// Key of logit x at index i: larger first, equal ones by lower index; 0 for none.
__device__ __forceinline__ uint32_t logit_order(float x) {
    if (!(x > -INFINITY)) return 0;  // -inf and NaN are no candidates
    const uint32_t bits = __float_as_uint(x == 0.0f ? 0.0f : x);
    return (bits & 0x80000000u) ? ~bits : (bits | 0x80000000u);
}
__device__ __forceinline__ uint64_t logit_key(float x, uint32_t i) {
    const uint32_t o = logit_order(x);
    return o ? ((uint64_t)o << 32) | (uint64_t)(0xFFFFFFFFu - i) : 0;
}
__device__ __forceinline__ float key_logit(uint64_t key) {
    const uint32_t o = (uint32_t)(key >> 32);
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}

__device__ __forceinline__ uint64_t lp_shfl_xor(uint64_t v, int m) {
    const unsigned lo = __shfl_xor((unsigned)v, m), hi = __shfl_xor((unsigned)(v >> 32), m);
    return ((uint64_t)hi << 32) | lo;
}
__device__ __forceinline__ uint64_t lp_max(uint64_t x, uint64_t y) { return x > y ? x : y; }

struct LpShared {
    uint64_t group[kLpGroups];
    uint32_t rank[kLpGroups];
    uint64_t cand[kLpCandidates];
    uint64_t top[kLpMaxK];
    uint64_t bound;
    uint64_t wave[kLpThreads / 64];
    uint32_t count;
    float red[3][kLpThreads / 64];
};

// The k largest of the workgroup's keys into sh.top, descending (0 where there
// are fewer). best: the thread's largest key; each(f) calls f on every key of the
// thread that may be among them.
template <typename EACH>
__device__ __forceinline__ void lp_select(LpShared& sh, unsigned k, uint64_t best, EACH&& each) {
    const unsigned t = threadIdx.x, lane = t & 63, wave = t >> 6;
    uint64_t g = lp_max(best, lp_shfl_xor(best, 1));  // groups of four threads
    g = lp_max(g, lp_shfl_xor(g, 2));
    if ((t & 3) == 0) sh.group[t >> 2] = g;
    if (t < kLpGroups) sh.rank[t] = 0;
    if (t < kLpMaxK) sh.top[t] = 0;
    if (t == 0) {
        sh.bound = 1;
        sh.count = 0;
    }
    __syncthreads();
    {
        const uint64_t mine = sh.group[lane];
        unsigned above = 0;
#pragma unroll
        for (unsigned i = 0; i < kLpGroups / 4; i++) above += sh.group[wave * (kLpGroups / 4) + i] > mine;
        atomicAdd(&sh.rank[lane], above);
    }
    __syncthreads();
    if (t < kLpGroups && sh.rank[t] == k - 1 && sh.group[t]) sh.bound = sh.group[t];
    __syncthreads();
    const uint64_t bound = sh.bound;
    if (best >= bound)
        each([&](uint64_t key) {
            if (key >= bound) {
                const unsigned at = atomicAdd(&sh.count, 1u);
                if (at < kLpCandidates) sh.cand[at] = key;
            }
        });
    __syncthreads();
    const unsigned n = sh.count;
    if (n <= kLpCandidates) {
        for (unsigned i = t; i < n; i += kLpThreads) {
            const uint64_t key = sh.cand[i];
            unsigned above = 0;
            for (unsigned j = 0; j < n; j++) above += sh.cand[j] > key;
            if (above < k) sh.top[above] = key;
        }
    } else {
        uint64_t last = ~0ull;
        for (unsigned r = 0; r < k; r++) {  // uniform
            uint64_t b = 0;
            each([&](uint64_t key) { b = key < last ? lp_max(b, key) : b; });
#pragma unroll
            for (int m = 32; m >= 1; m >>= 1) b = lp_max(b, lp_shfl_xor(b, m));
            if (lane == 0) sh.wave[wave] = b;
            __syncthreads();
            last = lp_max(lp_max(sh.wave[0], sh.wave[1]), lp_max(sh.wave[2], sh.wave[3]));
            if (t == 0) sh.top[r] = last;
            __syncthreads();
            if (!last) break;
        }
    }
    __syncthreads();
}

__device__ __forceinline__ float lp_wave_sum(float x) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) x += __shfl_xor(x, m);
    return x;
}
__device__ __forceinline__ float lp_wave_max(float x) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) x = fmaxf(x, __shfl_xor(x, m));
    return x;
}

// A row's results from its (m, S, U) and sh.top.
template <int DT>
__device__ __forceinline__ void lp_finish(const LogprobsArgs& a, const LpShared& sh, unsigned row, float m, float S, float U) {
    const unsigned t = threadIdx.x;
    const float none = __uint_as_float(0x7FC00000u);  // NaN
    const bool ok = S > 0.0f;                         // neither NaN nor empty
    const float logS = logf(S);
    if (t == 0) {
        if (a.entropy) a.entropy[row] = ok ? logS - U / S : none;
        if (a.logprobs) {
            const int32_t tok = a.tokens[row];
            float lp = 0.0f;
            if (tok >= 0 && (uint32_t)tok < a.vocab) {
                typedef typename LogitType<DT>::T T;
                const float x = logit_f32<DT>(static_cast<const T*>(a.logits)[row * a.row_stride + (uint32_t)tok]);
                lp = ok ? (logit_z(x, a) - m) - logS : none;
            }
            a.logprobs[row] = lp;
        }
    }
    if (t < a.k) {
        const uint64_t key = sh.top[t];
        a.top_ids[(uint64_t)row * a.k + t] = key ? (int32_t)(0xFFFFFFFFu - (uint32_t)key) : -1;
        a.top_logprobs[(uint64_t)row * a.k + t] =
            !ok ? none : key ? (logit_z(key_logit(key), a) - m) - logS : -INFINITY;
    }
}

// One chunk of one row. VEC: 16-byte loads (rows aligned), otherwise one element a load.
template <int DT, bool VEC>
__global__ __launch_bounds__(kLpThreads) void k_logprobs(const LogprobsArgs a) {
    typedef typename LogitType<DT>::T T;
    constexpr unsigned V = VEC ? 16 / sizeof(T) : 1;  // elements a load
    constexpr unsigned N = kLpElems / V;
    __shared__ LpShared sh;
    const unsigned t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const unsigned chunk = blockIdx.x, row = blockIdx.y;
    const unsigned i0 = chunk * kLpChunk;
    const T* src = static_cast<const T*>(a.logits) + row * a.row_stride;
    float x[kLpElems];
    if (i0 + kLpChunk <= a.vocab) {
        if constexpr (VEC) {
            u32x4 v[N];
#pragma unroll
            for (unsigned i = 0; i < N; i++)
                v[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(src + i0 + (i * kLpThreads + t) * V));
#pragma unroll
            for (unsigned i = 0; i < N; i++)
#pragma unroll
                for (unsigned e = 0; e < V; e++) {
                    if constexpr (sizeof(T) == 4) x[i * V + e] = __uint_as_float(v[i][e]);
                    else x[i * V + e] = logit_f32<DT>((uint16_t)(v[i][e / 2] >> (16 * (e & 1))));
                }
        } else {
#pragma unroll
            for (unsigned i = 0; i < kLpElems; i++) x[i] = logit_f32<DT>(src[i0 + i * kLpThreads + t]);
        }
    } else {
#pragma unroll
        for (unsigned i = 0; i < N; i++)
#pragma unroll
            for (unsigned e = 0; e < V; e++) {
                const unsigned at = i0 + (i * kLpThreads + t) * V + e;
                x[i * V + e] = at < a.vocab ? logit_f32<DT>(src[at]) : -INFINITY;
            }
    }

    float mx = -INFINITY;
    uint32_t mi = 0;  // the first place of the thread's maximum
#pragma unroll
    for (unsigned i = 0; i < kLpElems; i++) {
        if (x[i] > mx) {
            mx = x[i];
            mi = i;
        }
    }
    auto index_of = [&](unsigned i) __attribute__((always_inline)) { return i0 + (i / V * kLpThreads + t) * V + i % V; };
    const float wmax = lp_wave_max(mx);
    if (lane == 0) sh.red[0][wave] = wmax;
    __syncthreads();
    const float xmax = fmaxf(fmaxf(sh.red[0][0], sh.red[0][1]), fmaxf(sh.red[0][2], sh.red[0][3]));
    const float m = xmax == -INFINITY ? -INFINITY : logit_z(xmax, a);
    const float base = m == -INFINITY ? 0.0f : m;
    float S = 0.0f, U = 0.0f;
#pragma unroll
    for (unsigned i = 0; i < kLpElems; i++) {
        const float d = logit_z(x[i], a) - base;
        const float e = exp_f32(d);
        S += e;
        U += e == 0.0f ? 0.0f : d * e;
    }
    S = lp_wave_sum(S);
    U = lp_wave_sum(U);
    if (lane == 0) {
        sh.red[1][wave] = S;
        sh.red[2][wave] = U;
    }
    __syncthreads();
    S = (sh.red[1][0] + sh.red[1][1]) + (sh.red[1][2] + sh.red[1][3]);
    U = (sh.red[2][0] + sh.red[2][1]) + (sh.red[2][2] + sh.red[2][3]);
    if (a.k)
        lp_select(sh, a.k, logit_key(mx, index_of(mi)), [&](auto&& f) __attribute__((always_inline)) {
#pragma unroll
            for (unsigned i = 0; i < kLpElems; i++) f(logit_key(x[i], index_of(i)));
        });
    if (a.chunks == 1) {
        lp_finish<DT>(a, sh, row, m, S, U);
        return;
    }
    const uint64_t at = (uint64_t)row * a.chunks + chunk;
    if (t == 0) stg<f32x4>(a.part + at * 4, f32x4{m, S, U, 0.0f});
    if (t < a.k) a.cand[at * a.k + t] = sh.top[t];
}

// One row's chunks joined.
template <int DT>
__global__ __launch_bounds__(kLpThreads) void k_logprobs_join(const LogprobsArgs a) {
    __shared__ LpShared sh;
    const unsigned t = threadIdx.x, lane = t & 63, wave = t >> 6, row = blockIdx.x;
    const f32x4* part = reinterpret_cast<const f32x4*>(a.part) + (uint64_t)row * a.chunks;
    float m = -INFINITY;
    for (unsigned i = t; i < a.chunks; i += kLpThreads) m = fmaxf(m, part[i][0]);
    m = lp_wave_max(m);
    if (lane == 0) sh.red[0][wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(sh.red[0][0], sh.red[0][1]), fmaxf(sh.red[0][2], sh.red[0][3]));
    float S = 0.0f, U = 0.0f;
    for (unsigned i = t; i < a.chunks; i += kLpThreads) {
        const f32x4 p = part[i];
        if (p[0] == -INFINITY && !(p[1] != p[1])) continue;  // nothing in it (a NaN sum stays one)
        const float d = p[0] - m, f = exp_f32(d);
        S += p[1] * f;
        U += f == 0.0f ? 0.0f : (p[2] + d * p[1]) * f;
    }
    S = lp_wave_sum(S);
    U = lp_wave_sum(U);
    if (lane == 0) {
        sh.red[1][wave] = S;
        sh.red[2][wave] = U;
    }
    __syncthreads();
    S = (sh.red[1][0] + sh.red[1][1]) + (sh.red[1][2] + sh.red[1][3]);
    U = (sh.red[2][0] + sh.red[2][1]) + (sh.red[2][2] + sh.red[2][3]);
    if (a.k) {
        const uint64_t* cand = a.cand + (uint64_t)row * a.chunks * a.k;
        const unsigned n = a.chunks * a.k;
        uint64_t best = 0;
        for (unsigned i = t; i < n; i += kLpThreads) best = lp_max(best, cand[i]);
        lp_select(sh, a.k, best, [&](auto&& f) __attribute__((always_inline)) {
            for (unsigned i = t; i < n; i += kLpThreads) f(cand[i]);
        });
    }
    lp_finish<DT>(a, sh, row, m, S, U);
}

template <int DT>
void launch_logprobs(const LogprobsArgs& a, uint32_t rows, bool vec, hipStream_t st) {
    const dim3 grid(a.chunks, rows), block(kLpThreads);
    if (vec) G4_LAUNCH((k_logprobs<DT, true>), grid, block, 0, st, a);
    else G4_LAUNCH((k_logprobs<DT, false>), grid, block, 0, st, a);
    if (a.chunks > 1) G4_LAUNCH((k_logprobs_join<DT>), dim3(rows), block, 0, st, a);
}

}  // namespace g4

using namespace g4;

namespace {

int logprobs_check(const g4_token_logprobs_params* p, uint64_t* chunks) {
    if (!p) return fail(G4_EINVAL, "tokenLogprobs: NULL params");
    if (p->vocab == 0 || p->vocab > (1u << 24)) return fail(G4_EINVAL, "tokenLogprobs: vocab %u (1 to 2^24)", p->vocab);
    if (p->rows > 65535) return fail(G4_EINVAL, "tokenLogprobs: %u rows (at most 65535)", p->rows);
    if (p->top_k > kLpMaxK || p->top_k > p->vocab)
        return fail(G4_EINVAL, "tokenLogprobs: top_k %u (at most %u, and the vocab)", p->top_k, kLpMaxK);
    if (p->row_stride && p->row_stride < p->vocab)
        return fail(G4_EINVAL, "tokenLogprobs: row_stride below the vocab %u", p->vocab);
    if (p->row_stride > (1ull << 40)) return fail(G4_EINVAL, "tokenLogprobs: row_stride too long");
    if (p->dtype > G4_LOGITS_BF16) return fail(G4_EINVAL, "tokenLogprobs: dtype %u", p->dtype);
    if (!(p->cap >= 0.0f) || p->cap > 1e30f) return fail(G4_EINVAL, "tokenLogprobs: cap %g", (double)p->cap);
    if (!(p->temperature >= 1e-6f) || p->temperature > 1e6f)
        return fail(G4_EINVAL, "tokenLogprobs: temperature %g (1e-6 to 1e6)", (double)p->temperature);
    if (p->cap > 0.0f && p->cap < 1e-6f) return fail(G4_EINVAL, "tokenLogprobs: cap %g (0, or 1e-6 to 1e30)", (double)p->cap);
    *chunks = ((uint64_t)p->vocab + kLpChunk - 1) / kLpChunk;
    return G4_OK;
}

size_t logprobs_bytes(const g4_token_logprobs_params* p, uint64_t chunks) {
    return chunks == 1 ? 16 : (size_t)p->rows * chunks * (16 + 8ull * p->top_k) + 16;
}

}  // namespace

extern "C" {

int g4_token_logprobs_workspace_size(const g4_token_logprobs_params* p, size_t* bytes) {
    if (!bytes) return fail(G4_EINVAL, "g4_token_logprobs_workspace_size: bytes is NULL");
    uint64_t chunks = 0;
    const int rc = logprobs_check(p, &chunks);
    if (rc) return rc;
    *bytes = logprobs_bytes(p, chunks);
    return G4_OK;
}

int g4_token_logprobs(const void* logits, const int32_t* tokens, float* logprobs, float* entropy, int32_t* top_ids,
                      float* top_logprobs, const g4_token_logprobs_params* p, void* workspace, size_t workspace_bytes,
                      void* stream) {
    uint64_t chunks = 0;
    const int rc = logprobs_check(p, &chunks);
    if (rc) return rc;
    if (!logits || !workspace) return fail(G4_EINVAL, "tokenLogprobs: NULL logits or workspace");
    if (!tokens != !logprobs) return fail(G4_EINVAL, "tokenLogprobs: tokens and logprobs go together");
    if (!top_ids != !top_logprobs || !top_ids != (p->top_k == 0))
        return fail(G4_EINVAL, "tokenLogprobs: top_ids and top_logprobs go with a top_k above 0");
    if (!logprobs && !entropy && !top_ids) return fail(G4_EINVAL, "tokenLogprobs: nothing asked for");
    const size_t elem = p->dtype == G4_LOGITS_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(logits) & (elem - 1)) return fail(G4_EINVAL, "tokenLogprobs: misaligned logits");
    if (reinterpret_cast<uintptr_t>(workspace) & 15)
        return fail(G4_EINVAL, "tokenLogprobs: workspace must be 16-byte aligned");
    if (workspace_bytes < logprobs_bytes(p, chunks))
        return fail(G4_ENOSPC, "tokenLogprobs: workspace %zu bytes < %zu needed", workspace_bytes, logprobs_bytes(p, chunks));
    if (p->rows == 0) return G4_OK;
    LogprobsArgs a = {};
    a.logits = logits;
    a.tokens = tokens;
    a.logprobs = logprobs;
    a.entropy = entropy;
    a.top_ids = top_ids;
    a.top_logprobs = top_logprobs;
    a.part = static_cast<float*>(workspace);
    a.cand = reinterpret_cast<uint64_t*>(a.part + (uint64_t)p->rows * chunks * 4);
    a.row_stride = p->row_stride ? p->row_stride : p->vocab;
    a.vocab = p->vocab;
    a.chunks = (uint32_t)chunks;
    a.k = p->top_k;
    a.cap = p->cap;
    a.inv_cap = p->cap > 0.0f ? 1.0f / p->cap : 0.0f;
    a.temperature = p->temperature;
    a.inv_temperature = 1.0f / p->temperature;
    const bool vec = !((reinterpret_cast<uintptr_t>(logits) | (a.row_stride * elem)) & 15);
    hipStream_t st = as_stream(stream);
    if (p->dtype == G4_LOGITS_F32) launch_logprobs<G4_LOGITS_F32>(a, p->rows, vec, st);
    else if (p->dtype == G4_LOGITS_F16) launch_logprobs<G4_LOGITS_F16>(a, p->rows, vec, st);
    else launch_logprobs<G4_LOGITS_BF16>(a, p->rows, vec, st);
    G4_CHECK_LAUNCH("tokenLogprobs");
    return G4_OK;
}

}  // extern "C"
