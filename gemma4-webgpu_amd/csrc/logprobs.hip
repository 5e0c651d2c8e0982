// Log probabilities of given tokens, entropy and the best alternatives of rows
// of logits (g4_token_logprobs): what a step that verifies drafted tokens needs
// of them, next to the greedy head's argmax (lmhead.hip).
//
// z = cap tanh(x / cap) (or x), m = max z, t = (z - m) log2(e) / T, S = sum 2^t,
// U = sum t 2^t:  log p(i) = (t_i - log2 S) ln 2,  entropy = (log2 S - U / S) ln 2.
// Bound by the logits' bytes, read once: a workgroup takes a chunk of consecutive
// logits of a row into registers, so the maximum, the sums and the selection all
// work on what one pass has loaded. z is monotone in x, so maxima and ranks are
// taken on x itself and each element's z is evaluated once: one transcendental
// operation an element (three with a cap) and six plain ones (nine), which the
// loads of the other workgroups on a CU cover.
//
// Selection: candidates are 64-bit keys (order-preserving logit in the high half,
// inverted index in the low half), all different, so equal logits rank by index.
// The k-th largest of 64 groups' maxima bounds the k-th largest logit from below;
// the few logits at or above it are collected in LDS and ranked by counting. Where
// that bound lets too many through (logits in ascending order, or many equal
// ones), k rounds of a maximum below the last one take their place.
//
// Rows longer than a chunk leave (max x, S, U) and k keys per chunk in the workspace;
// a second launch, a workgroup a row, joins them in a fixed order.
//
// Measured at 262144 logits: 701 rows of 16 bits without alternatives 62 us, 5.9 TB/s (0.87 of
// a plain read stream); 64 rows of f32 with 20 alternatives 25 us, of which the second
// launch takes 5, and the selection, on workgroups that have all loaded and none left to
// load behind them, about 8; one row 10 us, two launches.
#include "decode_core.h"
#include "paged.h"

namespace g4 {

constexpr unsigned kLpThreads = 256;
constexpr unsigned kLpShort = 2048, kLpMiddle = 4096;  // logits of a chunk where rows are few: more workgroups,
                                                       // shorter chains
constexpr unsigned kLpLong = 8192;                     // and where they are many (twice as many logits of 16 bits)
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
    float* __restrict__ part;      // [rows][chunks][4]: max x, S, U
    uint64_t* __restrict__ cand;   // [rows][chunks][k]
    uint64_t row_stride;
    uint32_t vocab, chunks, k;
    float cap, cap_exp, cap_inv;  // and 2 log2(e) / cap, 1 / cap
    float slope;         // log2(e) / temperature
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

// cap tanh(x / cap). A mask of -inf stays one, and +inf too (it makes the row's sums NaN).
// Up to kLpNearCap as cap - 2 cap / (e^(2 x / cap) + 1), which is off by a few half-steps of the cap: 1e-5 at
// most, about what f32 logits near the cap are rounded by. Above it to a few half-steps of the value (half as
// many operations again).
constexpr float kLpNearCap = 64.0f;
template <bool NEAR>
__device__ __forceinline__ float logit_capped(float x, const LogprobsArgs& a) {
    float z;
    if constexpr (NEAR) {
        const float r = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * a.cap_exp) + 1.0f);
        z = __builtin_fmaf(-2.0f * a.cap, r, a.cap);
    } else {
        z = a.cap * tanh_f32(x * a.cap_inv);
    }
    return fabsf(x) == INFINITY ? x : z;
}
__device__ __forceinline__ float logit_z(float x, const LogprobsArgs& a) {
    if (a.cap > kLpNearCap) return logit_capped<false>(x, a);
    return a.cap > 0.0f ? logit_capped<true>(x, a) : x;
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
constexpr uint32_t kLpLeast = 0x00800000u;  // the lowest finite logit's order
__device__ __forceinline__ float order_logit(uint32_t o) { return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o); }
__device__ __forceinline__ float key_logit(uint64_t key) { return order_logit((uint32_t)(key >> 32)); }

__device__ __forceinline__ uint64_t lp_shfl_xor(uint64_t v, int m) {
    const unsigned lo = __shfl_xor((unsigned)v, m), hi = __shfl_xor((unsigned)(v >> 32), m);
    return ((uint64_t)hi << 32) | lo;
}
__device__ __forceinline__ uint64_t lp_max(uint64_t x, uint64_t y) { return x > y ? x : y; }

// Sum and maximum over the wave, in every lane: rotations of 16-lane rows, then rows and halves swapped.
template <int CTRL>
__device__ __forceinline__ float lp_dpp(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float lp_wave_sum(float x) {
    x += lp_dpp<0x128>(x);  // row_ror:8
    x += lp_dpp<0x124>(x);
    x += lp_dpp<0x122>(x);
    x += lp_dpp<0x121>(x);
    return add_xor32(add_xor16(x));
}
__device__ __forceinline__ float lp_wave_max(float x) {
    x = fmaxf(x, lp_dpp<0x128>(x));
    x = fmaxf(x, lp_dpp<0x124>(x));
    x = fmaxf(x, lp_dpp<0x122>(x));
    x = fmaxf(x, lp_dpp<0x121>(x));
    return max_xor32(max_xor16(x));
}

struct LpShared {
    uint32_t group[kLpGroups];
    uint64_t cand[kLpCandidates];
    uint64_t top[kLpMaxK];
    uint64_t wave[kLpThreads / 64];
    uint32_t count;
    float red[3][kLpThreads / 64];
};

// The selection of the k largest keys, in three steps with a barrier after each of the first two.
//
// Before the first barrier: best is the thread's largest logit, as its order.
__device__ __forceinline__ void lp_groups(LpShared& sh, uint32_t best) {
    const unsigned t = threadIdx.x;
    uint32_t g = max(best, (uint32_t)__builtin_amdgcn_mov_dpp((int)best, 0xB1, 0xf, 0xf, false));  // groups of four threads:
    g = max(g, (uint32_t)__builtin_amdgcn_mov_dpp((int)g, 0x4E, 0xf, 0xf, false));                 // quad_perm 1,0,3,2; 2,3,0,1
    if ((t & 3) == 0) sh.group[t >> 2] = g;
    if (t < kLpMaxK) sh.top[t] = 0;
    if (t == 0) sh.count = 0;
}
// After it: an order that at least k logits reach (kLpLeast where fewer are above -inf). The k-th largest of
// the 64 groups' maxima, bit by bit over the top 18 (sign, exponent, 9 of the fraction): each wave counts
// for itself.
__device__ __forceinline__ uint32_t lp_bound(const LpShared& sh, unsigned k) {
    const uint32_t mine = sh.group[threadIdx.x & 63];
    uint32_t bound = 0;
#pragma unroll
    for (int bit = 31; bit >= 14; bit--) {
        const uint32_t with = bound | 1u << bit;
        if ((unsigned)__popcll(__ballot(mine >= with)) >= k) bound = with;
    }
    return max(bound, kLpLeast);
}
// A thread's n keys into the candidates: put(f) calls f(key) for each.
template <typename PUT>
__device__ __forceinline__ void lp_push(LpShared& sh, unsigned n, PUT&& put) {
    if (n == 0) return;
    unsigned at = atomicAdd(&sh.count, n);
    put([&](uint64_t key) __attribute__((always_inline)) {
        if (at < kLpCandidates) sh.cand[at] = key;
        at++;
    });
}
// After the second barrier: store(rank, key) for the k largest, by the threads that have them; ranks there
// is no key for are left out. each(f) calls f on every key of the thread, should the candidates be too many.
template <typename STORE, typename EACH>
__device__ __forceinline__ void lp_rank(LpShared& sh, unsigned k, STORE&& store, EACH&& each) {
    const unsigned t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const unsigned n = sh.count;
    if (n <= kLpCandidates) {  // uniform
        for (unsigned i = t; i < n; i += kLpThreads) {
            const uint64_t key = sh.cand[i];
            unsigned above = 0;
            for (unsigned j = 0; j < n; j += 8) {  // eight reads at once
                uint64_t c[8];
#pragma unroll
                for (unsigned e = 0; e < 8; e++) c[e] = sh.cand[min(j + e, n - 1)];
#pragma unroll
                for (unsigned e = 0; e < 8; e++) above += j + e < n && c[e] > key;
            }
            if (above < k) store(above, key);
        }
        return;
    }
    uint64_t last = ~0ull;
    for (unsigned r = 0; r < k; r++) {  // uniform
        uint64_t b = 0;
        each([&](uint64_t key) __attribute__((always_inline)) { b = key < last ? lp_max(b, key) : b; });
#pragma unroll
        for (int m = 32; m >= 1; m >>= 1) b = lp_max(b, lp_shfl_xor(b, m));
        if (lane == 0) sh.wave[wave] = b;
        __syncthreads();
        last = lp_max(lp_max(sh.wave[0], sh.wave[1]), lp_max(sh.wave[2], sh.wave[3]));
        if (t == 0) store(r, last);
        __syncthreads();
        if (!last) break;
    }
}

// A row's results from its (max x, S, U) and sh.top.
template <int DT>
__device__ __forceinline__ void lp_finish(const LogprobsArgs& a, const LpShared& sh, unsigned row, float mx, float S, float U) {
    const unsigned t = threadIdx.x;
    constexpr float kLn2 = 0.69314718055994531f;
    const float none = __uint_as_float(0x7FC00000u);  // NaN
    const bool ok = S > 0.0f;                         // neither NaN nor empty
    const float m = logit_z(mx, a), logS = log2f(S);
    if (t == 0) {
        if (a.entropy) a.entropy[row] = ok ? (logS - U / S) * kLn2 : none;
        if (a.logprobs) {
            const int32_t tok = a.tokens[row];
            float lp = 0.0f;
            if (tok >= 0 && (uint32_t)tok < a.vocab) {
                typedef typename LogitType<DT>::T T;
                const float x = logit_f32<DT>(static_cast<const T*>(a.logits)[row * a.row_stride + (uint32_t)tok]);
                lp = ok ? ((logit_z(x, a) - m) * a.slope - logS) * kLn2 : none;
            }
            a.logprobs[row] = lp;
        }
    }
    if (t < a.k) {
        const uint64_t key = sh.top[t];
        a.top_ids[(uint64_t)row * a.k + t] = key ? (int32_t)(0xFFFFFFFFu - (uint32_t)key) : -1;
        a.top_logprobs[(uint64_t)row * a.k + t] =
            !ok ? none : key ? ((logit_z(key_logit(key), a) - m) * a.slope - logS) * kLn2 : -INFINITY;
    }
}

// One chunk of one row, E logits a thread. VEC: 16-byte loads (rows aligned), otherwise one element a load.
template <int DT, bool VEC, int E>
__global__ __launch_bounds__(kLpThreads, E <= 32 ? 4 : 3) void k_logprobs(const LogprobsArgs a) {
    typedef typename LogitType<DT>::T T;
    constexpr int V = VEC ? 16 / sizeof(T) : 1;  // elements a load
    constexpr int N = E / V, P = sizeof(T) == 2 ? 2 : 1;  // logits a register
    static_assert(E % V == 0 && E % P == 0, "whole loads and registers");
    __shared__ LpShared sh;
    const unsigned t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const unsigned chunk = blockIdx.x, row = blockIdx.y;
    const unsigned i0 = chunk * (kLpThreads * E);
    const T* src = static_cast<const T*>(a.logits) + row * a.row_stride;
    uint32_t raw[E / P];
    auto index_of = [&](int i) __attribute__((always_inline)) { return i0 + (i / V * kLpThreads + t) * V + i % V; };
    auto logit = [&](int i) __attribute__((always_inline)) -> float {  // i: a constant
        if constexpr (P == 1) return __uint_as_float(raw[i]);
        else return logit_f32<DT>((T)(raw[i / 2] >> (16 * (i & 1))));
    };
    if (i0 + kLpThreads * E <= a.vocab) {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < N; i++) {
                const u32x4 v = ldg_stream<u32x4>(src + i0 + (i * kLpThreads + t) * V);
#pragma unroll
                for (int e = 0; e < 4; e++) raw[4 * i + e] = v[e];
            }
        } else {
            T v[E];
#pragma unroll
            for (int i = 0; i < E; i++) v[i] = src[index_of(i)];
#pragma unroll
            for (int i = 0; i < E; i += P) {
                if constexpr (P == 1) raw[i] = __builtin_bit_cast(uint32_t, v[i]);
                else raw[i / 2] = (uint32_t)v[i] | (uint32_t)v[i + 1] << 16;
            }
        }
    } else {
        const T none = P == 1 ? (T)-INFINITY : DT == G4_LOGITS_F16 ? (T)0xFC00 : (T)0xFF80;  // -inf
        T v[E];
#pragma unroll
        for (int i = 0; i < E; i++) v[i] = index_of(i) < a.vocab ? src[index_of(i)] : none;
#pragma unroll
        for (int i = 0; i < E; i += P) {
            if constexpr (P == 1) raw[i] = __builtin_bit_cast(uint32_t, v[i]);
            else raw[i / 2] = (uint32_t)v[i] | (uint32_t)v[i + 1] << 16;
        }
    }

    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < E; i++) mx = fmaxf(mx, logit(i));  // leaves NaN aside
    const float wmax = lp_wave_max(mx);
    if (lane == 0) sh.red[0][wave] = wmax;
    if (a.k) lp_groups(sh, logit_order(mx));
    __syncthreads();
    const float xmax = fmaxf(fmaxf(sh.red[0][0], sh.red[0][1]), fmaxf(sh.red[0][2], sh.red[0][3]));
    const float m = xmax == -INFINITY ? 0.0f : logit_z(xmax, a);
    float S = 0.0f, U = 0.0f;
    // 2^t is 0 from -200 on, where t 2^t must not become -inf times 0; a NaN goes on in S.
    auto sums = [&](auto&& z) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < E; i++) {
            const float d = (z(logit(i)) - m) * a.slope, e = __builtin_amdgcn_exp2f(d);
            S += e;
            U = __builtin_fmaf(e, fmaxf(d, -200.0f), U);
        }
    };
    if (a.cap > kLpNearCap) sums([&](float x) __attribute__((always_inline)) { return logit_capped<false>(x, a); });
    else if (a.cap > 0.0f) sums([&](float x) __attribute__((always_inline)) { return logit_capped<true>(x, a); });
    else sums([](float x) __attribute__((always_inline)) { return x; });
    S = lp_wave_sum(S);
    U = lp_wave_sum(U);
    if (lane == 0) {
        sh.red[1][wave] = S;
        sh.red[2][wave] = U;
    }
    if (a.k) {
        const float least = order_logit(lp_bound(sh, a.k));
        unsigned n = 0;
        if (mx >= least) {
#pragma unroll
            for (int i = 0; i < E; i++) n += logit(i) >= least;  // neither NaN nor -inf
        }
        lp_push(sh, n, [&](auto&& f) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < E; i++)
                if (logit(i) >= least) f(logit_key(logit(i), index_of(i)));
        });
    }
    __syncthreads();
    S = (sh.red[1][0] + sh.red[1][1]) + (sh.red[1][2] + sh.red[1][3]);
    U = (sh.red[2][0] + sh.red[2][1]) + (sh.red[2][2] + sh.red[2][3]);
    auto each = [&](auto&& f) __attribute__((always_inline)) {
        // Computed where it stands: kept for the next round, the keys would take the registers of the common path.
        float zero = 0.0f;
        asm volatile("" : "+v"(zero));
#pragma unroll
        for (int i = 0; i < E; i++) f(logit_key(logit(i) + zero, index_of(i)));
    };
    if (a.chunks == 1) {
        if (a.k) {
            lp_rank(sh, a.k, [&](unsigned r, uint64_t key) __attribute__((always_inline)) { sh.top[r] = key; }, each);
            __syncthreads();
        }
        lp_finish<DT>(a, sh, row, xmax, S, U);
        return;
    }
    const uint64_t at = (uint64_t)row * a.chunks + chunk;
    if (t == 0) stg<f32x4>(a.part + at * 4, f32x4{xmax, S, U, 0.0f});
    if (a.k) {
        uint64_t* dst = a.cand + at * a.k;
        const unsigned n = sh.count;
        if (n < a.k && t >= n && t < a.k) dst[t] = 0;  // fewer above -inf
        lp_rank(sh, a.k, [&](unsigned r, uint64_t key) __attribute__((always_inline)) { dst[r] = key; }, each);
    }
}

// One row's chunks joined.
template <int DT>
__global__ __launch_bounds__(kLpThreads) void k_logprobs_join(const LogprobsArgs a) {
    __shared__ LpShared sh;
    const unsigned t = threadIdx.x, lane = t & 63, wave = t >> 6, row = blockIdx.x;
    const f32x4* part = reinterpret_cast<const f32x4*>(a.part) + (uint64_t)row * a.chunks;
    const uint64_t* cand = a.cand + (uint64_t)row * a.chunks * a.k;
    const unsigned n = a.chunks * a.k;
    constexpr unsigned H = 4;  // keys a thread holds; more are read again
    uint64_t held[H];
    uint64_t best = 0;
#pragma unroll
    for (unsigned i = 0; i < H; i++) held[i] = t + i * kLpThreads < n ? cand[t + i * kLpThreads] : 0;
    const f32x4 p0 = t < a.chunks ? part[t] : f32x4{-INFINITY, 0.0f, 0.0f, 0.0f};
    float mx = p0[0];
    for (unsigned i = t + kLpThreads; i < a.chunks; i += kLpThreads) mx = fmaxf(mx, part[i][0]);
    mx = lp_wave_max(mx);
    if (lane == 0) sh.red[0][wave] = mx;
    if (a.k) {
#pragma unroll
        for (unsigned i = 0; i < H; i++) best = lp_max(best, held[i]);
        for (unsigned i = t + H * kLpThreads; i < n; i += kLpThreads) best = lp_max(best, cand[i]);
        lp_groups(sh, (uint32_t)(best >> 32));
    }
    __syncthreads();
    mx = fmaxf(fmaxf(sh.red[0][0], sh.red[0][1]), fmaxf(sh.red[0][2], sh.red[0][3]));
    const float m = mx == -INFINITY ? 0.0f : logit_z(mx, a);
    float S = 0.0f, U = 0.0f;
    auto add = [&](const f32x4& p) __attribute__((always_inline)) {
        const float d = (p[0] == -INFINITY ? 0.0f : logit_z(p[0], a) - m) * a.slope;  // of an empty chunk: S is 0 or NaN
        const float f = __builtin_amdgcn_exp2f(d);
        S += p[1] * f;
        U += f == 0.0f ? 0.0f : (p[2] + d * p[1]) * f;
    };
    add(p0);
    for (unsigned i = t + kLpThreads; i < a.chunks; i += kLpThreads) add(part[i]);
    S = lp_wave_sum(S);
    U = lp_wave_sum(U);
    if (lane == 0) {
        sh.red[1][wave] = S;
        sh.red[2][wave] = U;
    }
    auto each = [&](auto&& f) __attribute__((always_inline)) {
#pragma unroll
        for (unsigned i = 0; i < H; i++) f(held[i]);
        for (unsigned i = t + H * kLpThreads; i < n; i += kLpThreads) f(cand[i]);
    };
    if (a.k) {
        const uint32_t bound = lp_bound(sh, a.k);
        unsigned many = 0;
        if ((uint32_t)(best >> 32) >= bound)
            each([&](uint64_t key) __attribute__((always_inline)) { many += (uint32_t)(key >> 32) >= bound; });
        lp_push(sh, many, [&](auto&& f) __attribute__((always_inline)) {
            each([&](uint64_t key) __attribute__((always_inline)) {
                if ((uint32_t)(key >> 32) >= bound) f(key);
            });
        });
    }
    __syncthreads();
    S = (sh.red[1][0] + sh.red[1][1]) + (sh.red[1][2] + sh.red[1][3]);
    U = (sh.red[2][0] + sh.red[2][1]) + (sh.red[2][2] + sh.red[2][3]);
    if (a.k) {
        lp_rank(sh, a.k, [&](unsigned r, uint64_t key) __attribute__((always_inline)) { sh.top[r] = key; }, each);
        __syncthreads();
    }
    lp_finish<DT>(a, sh, row, mx, S, U);
}

// Long chunks where they fill the chip twice; else shorter ones, as long as a row has at most 64 for the second
// launch to join. (Chunks of 2048 / 4096 / 8192 logits: a row of 50257 10.4 / 11.7 / 13.5 us, one of 262144
// 12.6 / 10.8 / 11.8, 64 of those 33.8 / 25.5 / 24.8.)
static uint32_t lp_chunk(uint32_t rows, uint32_t vocab) {
    if ((uint64_t)rows * ((vocab + kLpLong - 1) / kLpLong) >= 2 * (uint64_t)device_cus()) return kLpLong;
    return vocab <= 64 * kLpShort ? kLpShort : kLpMiddle;
}
static uint64_t lp_chunks(uint32_t rows, uint32_t vocab) {
    const uint64_t chunk = lp_chunk(rows, vocab);
    return (vocab + chunk - 1) / chunk;
}
// The most chunks that a call of at most this many rows and logits has, all rows together: fewer rows or logits may
// be cut shorter. Cut long, a call has at most rows * long; cut short, fewer than 2 CUs long chunks' worth of logits
// (or it would be cut long), of four short chunks each.
static uint64_t lp_most_chunks(uint32_t rows, uint32_t vocab) {
    const uint64_t longs = (vocab + kLpLong - 1) / kLpLong, middles = (vocab + kLpMiddle - 1) / kLpMiddle;
    const uint64_t shorts = vocab <= 64 * kLpShort ? (vocab + kLpShort - 1) / kLpShort : 64;
    const uint64_t cut_short = rows * (shorts > middles ? shorts : middles), least = 8ull * (uint64_t)device_cus();
    return cut_short <= least ? cut_short : rows * longs > least ? rows * longs : least;
}

template <int DT, int E>
void launch_chunks(const LogprobsArgs& a, uint32_t rows, bool vec, hipStream_t st) {
    const dim3 grid(a.chunks, rows), block(kLpThreads);
    if (vec) G4_LAUNCH((k_logprobs<DT, true, E>), grid, block, 0, st, a);
    else G4_LAUNCH((k_logprobs<DT, false, E>), grid, block, 0, st, a);
}

template <int DT>
void launch_logprobs(LogprobsArgs& a, uint32_t rows, bool vec, hipStream_t st) {
    constexpr int P = DT == G4_LOGITS_F32 ? 1 : 2;
    const uint32_t least = lp_chunk(rows, a.vocab), chunk = least == kLpLong ? kLpLong * P : least;
    a.chunks = (a.vocab + chunk - 1) / chunk;
    a.cand = reinterpret_cast<uint64_t*>(a.part + (uint64_t)rows * a.chunks * 4);
    if (least == kLpShort) launch_chunks<DT, kLpShort / kLpThreads>(a, rows, vec, st);
    else if (least == kLpMiddle) launch_chunks<DT, kLpMiddle / kLpThreads>(a, rows, vec, st);
    else launch_chunks<DT, kLpLong * P / kLpThreads>(a, rows, vec, st);
    if (a.chunks > 1) G4_LAUNCH((k_logprobs_join<DT>), dim3(rows), dim3(kLpThreads), 0, st, a);
}

}  // namespace g4

using namespace g4;

namespace {

int logprobs_check(const g4_token_logprobs_params* p) {
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
    return G4_OK;
}

// Room for so many chunks, of any type and alignment.
size_t logprobs_bytes(const g4_token_logprobs_params* p, uint64_t chunks) {
    return (size_t)chunks * (16 + 8ull * p->top_k) + 16;
}

}  // namespace

extern "C" {

int g4_token_logprobs_workspace_size(const g4_token_logprobs_params* p, size_t* bytes) {
    if (!bytes) return fail(G4_EINVAL, "g4_token_logprobs_workspace_size: bytes is NULL");
    const int rc = logprobs_check(p);
    if (rc) return rc;
    *bytes = logprobs_bytes(p, lp_most_chunks(p->rows, p->vocab));
    return G4_OK;
}

int g4_token_logprobs(const void* logits, const int32_t* tokens, float* logprobs, float* entropy, int32_t* top_ids,
                      float* top_logprobs, const g4_token_logprobs_params* p, void* workspace, size_t workspace_bytes,
                      void* stream) {
    const int rc = logprobs_check(p);
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
    const size_t need = logprobs_bytes(p, p->rows * lp_chunks(p->rows, p->vocab));
    if (workspace_bytes < need)
        return fail(G4_ENOSPC, "tokenLogprobs: workspace %zu bytes < %zu needed", workspace_bytes, need);
    if (p->rows == 0) return G4_OK;
    LogprobsArgs a = {};
    a.logits = logits;
    a.tokens = tokens;
    a.logprobs = logprobs;
    a.entropy = entropy;
    a.top_ids = top_ids;
    a.top_logprobs = top_logprobs;
    a.part = static_cast<float*>(workspace);
    a.row_stride = p->row_stride ? p->row_stride : p->vocab;
    a.vocab = p->vocab;
    a.k = p->top_k;
    a.cap = p->cap;
    a.cap_exp = p->cap > 0.0f ? 2.0f * kLog2e / p->cap : 0.0f;
    a.cap_inv = p->cap > 0.0f ? 1.0f / p->cap : 0.0f;
    a.slope = kLog2e / p->temperature;
    const bool vec = !((reinterpret_cast<uintptr_t>(logits) | (a.row_stride * elem)) & 15);
    hipStream_t st = as_stream(stream);
    if (p->dtype == G4_LOGITS_F32) launch_logprobs<G4_LOGITS_F32>(a, p->rows, vec, st);
    else if (p->dtype == G4_LOGITS_F16) launch_logprobs<G4_LOGITS_F16>(a, p->rows, vec, st);
    else launch_logprobs<G4_LOGITS_BF16>(a, p->rows, vec, st);
    G4_CHECK_LAUNCH("tokenLogprobs");
    return G4_OK;
}

}  // extern "C"
