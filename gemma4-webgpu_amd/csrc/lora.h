// Low-rank adapters of many requests at once, as the kernels see them (lora.hip,
// linear8.hip): token t has adapter ids[t], or none where that is not in
// [0, n_adapters).
//
// Two products. Down: u[t][i] = sum_k x[t][k] A[a][i][k], i over the segments' rank rows each,
// left in the workspace in f32 (lora.hip). Up, here, as an epilogue of whatever made the token's
// outputs: acc[o] += scale[a] sum_j u[s(o)][j] B[a][o][j].
//
// Where a tile's tokens share an adapter or two, the up product runs on the 16-bit MFMA: u enters as the f16 parts of u 2^e (2^e: the token's
// largest |u| comes to lie in [2^14, 2^15)) and of what the first leaves, off by 2^-23 of itself or 2^-39
// of the largest; with bf16 adapters as three bf16 parts, off by 2^-25. f32 products take eight times the cycles.
// Where they have more, an adapter after the other would wait for memory each time (64 requests of 40 adapters: 43 us);
// then every lane takes its own token's rows and adds the products in f32, all loads independent of each other.
#pragma once

#include "decode_core.h"
#include "rows.h"

namespace g4 {

constexpr unsigned kLoraMaxRank = 128;

struct LoraDev {
    const void* __restrict__ a;        // [n_adapters][down][n]
    const void* __restrict__ b;        // [n_adapters][rows][rank]
    const float* __restrict__ scales;  // [n_adapters] or nullptr: 1
    const int32_t* __restrict__ ids;   // [n_tokens]
    float* __restrict__ u;             // [n_tokens][down]
    uint32_t n_adapters, rank, n, n_segs;
    uint32_t ends[4];                  // of the segments' outputs; those past n_segs as the last
    uint32_t rows, down;               // outputs; n_segs * rank
    uint32_t n_tokens;
};

__device__ __forceinline__ int lora_id(const LoraDev& l, unsigned t, bool valid) {
    const int id = valid ? l.ids[t] : -1;
    return (unsigned)id < l.n_adapters ? id : -1;
}

// The up product's tile: M outputs by M tokens. A lane holds, of token column lane % M, outputs 4 group + i % 4 + 8 (i / 4)
// with M 32, 4 group + i with M 16, where group = lane / M; its operands hold eight j of every STEP from 8 group on.
template <int M>
struct LoraTile;
template <>
struct LoraTile<16> {
    typedef f32x4 acc;
    static constexpr unsigned STEP = 32;
    static __device__ __forceinline__ acc mfma(f16x8 a, f16x8 b, acc c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ acc mfma(bf16x8 a, bf16x8 b, acc c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ float most(float x) { return max_xor32(max_xor16(x)); }
};
template <>
struct LoraTile<32> {
    typedef f32x16 acc;
    static constexpr unsigned STEP = 16;
    static __device__ __forceinline__ acc mfma(f16x8 a, f16x8 b, acc c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ acc mfma(bf16x8 a, bf16x8 b, acc c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ float most(float x) { return max_xor32(x); }
};

// Adapters of a tile that are taken one after the other (us of lora_add, 64 tokens, n 1536, one after the other / by lane: rank
// 16, two a tile 7.0 / 6.0, four 8.8 / 5.9, eight 12.5 / 6.1; rank 64, one 6.7 / 8.3, two 7.7 / 8.3, four 9.8 / 8.3).
constexpr int kLoraShared = 2;

template <bool BF>
__device__ __forceinline__ float lora_dot8(u32x4 w, f32x4 x, f32x4 y, float sum) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float lo = BF ? __uint_as_float(w[i] << 16) : h2f((uint16_t)w[i]), hi = BF ? __uint_as_float(w[i] & 0xFFFF0000u) : h2f((uint16_t)(w[i] >> 16));
        sum = __builtin_fmaf(lo, i < 2 ? x[2 * i] : y[2 * i - 4], sum);
        sum = __builtin_fmaf(hi, i < 2 ? x[2 * i + 1] : y[2 * i - 3], sum);
    }
    return sum;
}

// Adds a column tile's adapters to NRT row tiles of outputs from o0 on, through add(rt, i, value) for each element of the
// lane's: token `t` of column lane % M, its adapter `id`, -1 none. BF: bf16 adapters. AHEAD: more operands are
// requested at once, where the registers allow it.
template <int M, int NRT, bool BF, bool AHEAD = true, typename ADD>
__device__ __forceinline__ void lora_up(const LoraDev& l, unsigned o0, unsigned t, int id, ADD&& add) {
    using T = LoraTile<M>;
    constexpr int N = sizeof(typename T::acc) / 4;
    unsigned lane = threadIdx.x & 63;
    if constexpr (M == 32) asm volatile("" : "+v"(lane));  // what follows from it is not kept from call to call
    const unsigned col = lane % M, g = lane / M;
    uint64_t left = __ballot(id >= 0);
    int others = 0;
    for (uint64_t rest = left; rest && others <= kLoraShared; others++)  // uniform, as all below
        rest &= ~__ballot(id == __builtin_amdgcn_readlane(id, __builtin_ctzll(rest)));
    if (others > kLoraShared) {
        const float alpha = id < 0 ? 0.0f : l.scales ? l.scales[id] : 1.0f;
        const uint16_t* b = static_cast<const uint16_t*>(l.b) + (uint64_t)max(id, 0) * l.rows * l.rank;
        unsigned first = 0;
#pragma unroll 1
        for (unsigned s = 0; s < l.n_segs; s++) {
            const unsigned end = l.ends[s];
            if (end > o0 && first < o0 + M * NRT) {
                const float* u = l.u + (uint64_t)t * l.down + s * l.rank;
                constexpr int P = AHEAD ? 4 : 2;  // outputs at a time
#pragma unroll
                for (int q = 0; q < NRT * N / P; q++) {
                    const int rt = P * q / N, i = P * q % N;
                    const unsigned o = o0 + M * rt + 8 * (i / 4) + 4 * g + i % 4;
                    float sum[P] = {};
                    const bool some = id >= 0 && o < end && o + P > first;
#pragma unroll AHEAD ? 2 : 1
                    for (unsigned j = 0; j < l.rank; j += 8) {
                        if (!some) continue;
                        const f32x4 x = ldg<f32x4>(u + j), y = ldg<f32x4>(u + j + 4);
                        u32x4 w[P];
#pragma unroll
                        for (int e = 0; e < P; e++) w[e] = ldg<u32x4>(b + (uint64_t)min(o + e, l.rows - 1) * l.rank + j);
#pragma unroll
                        for (int e = 0; e < P; e++) sum[e] = lora_dot8<BF>(w[e], x, y, sum[e]);
                    }
#pragma unroll
                    for (int e = 0; e < P; e++)
                        if (some && o + e >= first && o + e < end) add(rt, i + e, sum[e] * alpha);
                    if constexpr (!AHEAD) __builtin_amdgcn_sched_barrier(0);
                }
            }
            first = end;
        }
        return;
    }
    while (left) {  // an adapter of the tile at a time
        const int a = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
        left &= ~__ballot(id == a);
        const bool mine = id == a;
        const float alpha = l.scales ? l.scales[a] : 1.0f;
        const uint16_t* b = static_cast<const uint16_t*>(l.b) + (uint64_t)a * l.rows * l.rank;
        unsigned first = 0;
#pragma unroll 1
        for (unsigned s = 0; s < l.n_segs; s++) {
            const unsigned end = l.ends[s];
            if (end > o0 && first < o0 + M * NRT) {
                const unsigned steps = (l.rank + T::STEP - 1) / T::STEP;
                const float* u = l.u + (uint64_t)t * l.down + s * l.rank + 8 * g;
                typename T::acc d[NRT];
#pragma unroll
                for (int rt = 0; rt < NRT; rt++)
#pragma unroll
                    for (int i = 0; i < N; i++) d[rt][i] = 0.0f;
                struct Ops {
                    f32x4 x, y;
                    u32x4 w[NRT];
                };
                constexpr unsigned BATCH = AHEAD ? 4 : 1;  // steps whose operands are requested at once
                auto fetch = [&](unsigned st) __attribute__((always_inline)) {
                    const unsigned j = T::STEP * st + 8 * g;
                    f32x4 x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
                    if (mine && j < l.rank) {
                        x = ldg<f32x4>(u + T::STEP * st);
                        y = ldg<f32x4>(u + T::STEP * st + 4);
                    }
                    Ops r;
                    r.x = x;
                    r.y = y;
#pragma unroll
                    for (int rt = 0; rt < NRT; rt++) {
                        const unsigned o = o0 + M * rt + col;
                        u32x4 w = {0, 0, 0, 0};
                        if (o >= first && o < end && j < l.rank) w = ldg<u32x4>(b + (uint64_t)o * l.rank + j);
                        r.w[rt] = w;
                    }
                    return r;
                };
                auto most = [](float m, const f32x4& x, const f32x4& y) __attribute__((always_inline)) {
#pragma unroll
                    for (int i = 0; i < 4; i++) m = fmaxf(m, fmaxf(fabsf(x[i]), fabsf(y[i])));
                    return m;
                };
                float up = 1.0f, down = 1.0f;
#pragma unroll 1
                for (unsigned st0 = 0; st0 < steps; st0 += BATCH) {
                    Ops ops[BATCH];
#pragma unroll
                    for (unsigned i = 0; i < BATCH; i++) ops[i] = fetch(st0 + i);  // past the last: zeros
                    if (!BF && st0 == 0) {  // the token's largest, of these and of the others
                        float m = 0.0f;
#pragma unroll
                        for (unsigned i = 0; i < BATCH; i++) m = most(m, ops[i].x, ops[i].y);
#pragma unroll 2
                        for (unsigned st = BATCH; st < steps; st++) {
                            f32x4 x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
                            if (mine && T::STEP * st + 8 * g < l.rank) {
                                x = ldg<f32x4>(u + T::STEP * st);
                                y = ldg<f32x4>(u + T::STEP * st + 4);
                            }
                            m = most(m, x, y);
                        }
                        const unsigned e = max(__float_as_uint(T::most(m)) >> 23, 15u);
                        up = __uint_as_float((268u - e) << 23);
                        down = __uint_as_float((e - 14u) << 23);
                    }
#pragma unroll
                    for (unsigned b4 = 0; b4 < BATCH; b4++) {
                        const Ops& now = ops[b4];
                        if (st0 + b4 >= steps) continue;
                        float x[8];
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            x[i] = now.x[i] * up;
                            x[4 + i] = now.y[i] * up;
                        }
                        if constexpr (BF) {
                            bf16x8 p0, p1, p2;
#pragma unroll
                            for (int i = 0; i < 8; i++) {
                                p0[i] = (__bf16)x[i];
                                const float r = x[i] - (float)p0[i];
                                p1[i] = (__bf16)r;
                                p2[i] = (__bf16)(r - (float)p1[i]);
                            }
#pragma unroll
                            for (int rt = 0; rt < NRT; rt++) {
                                const bf16x8 wb = __builtin_bit_cast(bf16x8, now.w[rt]);
                                d[rt] = T::mfma(wb, p2, d[rt]);
                                d[rt] = T::mfma(wb, p1, d[rt]);
                                d[rt] = T::mfma(wb, p0, d[rt]);
                            }
                        } else {
                            f16x8 p0, p1;
#pragma unroll
                            for (int i = 0; i < 8; i++) {
                                p0[i] = (f16)x[i];
                                p1[i] = (f16)(x[i] - (float)p0[i]);
                            }
#pragma unroll
                            for (int rt = 0; rt < NRT; rt++) {
                                const f16x8 wh = __builtin_bit_cast(f16x8, now.w[rt]);
                                d[rt] = T::mfma(wh, p1, d[rt]);
                                d[rt] = T::mfma(wh, p0, d[rt]);
                            }
                        }
                    }
                }
                const float f = down * alpha;
                if (o0 >= first && o0 + M * NRT <= end) {
#pragma unroll
                    for (int rt = 0; rt < NRT; rt++) {
#pragma unroll
                        for (int i = 0; i < N; i++)
                            if (mine) add(rt, i, d[rt][i] * f);
                    }
                } else {
                    // Outputs of the tile's other segments: sums of zero weights, which an Inf or NaN among u makes NaN.
                    const unsigned before = first - (o0 + 4 * g), width = mine ? end - first : 0;
#pragma unroll
                    for (int rt = 0; rt < NRT; rt++) {
#pragma unroll
                        for (int i = 0; i < N; i++)
                            if (M * rt + 8 * (i / 4) + i % 4 - before < width) add(rt, i, d[rt][i] * f);
                    }
                }
            }
            first = end;
        }
    }
}

// What the up product reads beside its base, and what the down product does beside x and its scales.
struct LoraOperands {
    Operand a, b, scales, ids, u;
};
inline LoraOperands lora_operands(const LoraDev& d) {
    const uint64_t L = d.n_adapters;
    return {{"the adapters' down rows", one_range(d.a, L * d.down * d.n * 2)},
            {"the adapters' up rows", one_range(d.b, L * d.rows * d.rank * 2)},
            {"the adapters' scales", one_range(d.scales, L * 4)},
            {"adapter_ids", one_range(d.ids, (uint64_t)d.n_tokens * 4)},
            {"workspace", one_range(d.u, (uint64_t)d.n_tokens * d.down * 4)}};
}

// The description checked and brought into the kernels' form; `what` names the call.
int lora_check(const char* what, const g4_lora* l);
LoraDev lora_dev(const g4_lora* l, uint32_t n_tokens);
size_t lora_bytes(const g4_lora* l, uint32_t n_tokens);  // of u
// The down product of every token that has an adapter; d.u and d.ids set. x: rows of x_type, x_scales with e4m3.
void lora_launch_down(const LoraDev& d, uint32_t lora_type, const void* x, uint32_t x_type, uint64_t x_stride,
                      const float* x_scales, hipStream_t st);

}  // namespace g4
