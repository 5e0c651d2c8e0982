// Low-rank adapters of many requests at once, as the kernels see them (lora.hip,
// linear8.hip): token t has adapter ids[t], or none where that is not in
// [0, n_adapters).
//
// Two products. Down: u[t][i] = sum_k x[t][k] A[a][i][k], i over the segments' rank rows each,
// left in the workspace as f32 partial sums of pieces of k (lora.hip). Up, here, as an
// epilogue of whatever made the token's outputs: acc[o] += scale[a] sum_j u[s(o)][j] B[a][o][j].
//
// The up product runs on the 16-bit MFMA: u enters as the f16 parts of u 2^e (2^e: the token's
// largest |u| comes to lie in [2^14, 2^15)) and of what the first leaves, off by 2^-23 of itself or 2^-39
// of the largest; with bf16 adapters as three bf16 parts, off by 2^-25. f32 products take eight times the cycles.
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
    float* __restrict__ u;             // [splits][n_tokens][down]
    uint32_t n_adapters, rank, n, n_segs;
    uint32_t ends[4];                  // of the segments' outputs; those past n_segs as the last
    uint32_t rows, down;               // outputs; n_segs * rank
    uint32_t splits, n_tokens;
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

// Adds a column tile's adapters to NRT row tiles of outputs from o0 on, through add(rt, i, value) for each element of the
// lane's: token `t` of column lane % M, its adapter `id`, -1 none. BF: bf16 adapters.
template <int M, int NRT, bool BF, typename ADD>
__device__ __forceinline__ void lora_up(const LoraDev& l, unsigned o0, unsigned t, int id, ADD&& add) {
    using T = LoraTile<M>;
    constexpr int N = sizeof(typename T::acc) / 4;
    const unsigned lane = threadIdx.x & 63, col = lane % M, g = lane / M;
    uint64_t left = __ballot(id >= 0);
    while (left) {  // an adapter of the tile at a time; uniform
        const int a = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
        left &= ~__ballot(id == a);
        const bool mine = id == a;
        const float alpha = l.scales ? l.scales[a] : 1.0f;
        const uint16_t* b = static_cast<const uint16_t*>(l.b) + (uint64_t)a * l.rows * l.rank;
        unsigned first = 0;
#pragma unroll 1
        for (unsigned s = 0; s < l.n_segs; s++) {  // uniform
            const unsigned end = l.ends[s];
            if (end > o0 && first < o0 + M * NRT) {
                const unsigned steps = (l.rank + T::STEP - 1) / T::STEP;
                typename T::acc d[NRT];
#pragma unroll
                for (int rt = 0; rt < NRT; rt++)
#pragma unroll
                    for (int i = 0; i < N; i++) d[rt][i] = 0.0f;
                const float* u = l.u + (uint64_t)t * l.down + s * l.rank;
                const uint64_t piece = (uint64_t)l.n_tokens * l.down;
                auto part = [&](unsigned j) __attribute__((always_inline)) {  // u[j .. j + 8)
                    struct { f32x4 a, b; } v = {{0, 0, 0, 0}, {0, 0, 0, 0}};
                    if (mine && j < l.rank) {
                        for (unsigned p = 0; p < l.splits; p++) {
                            v.a += ldg<f32x4>(u + p * piece + j);
                            v.b += ldg<f32x4>(u + p * piece + j + 4);
                        }
                    }
                    return v;
                };
                float up = 1.0f, down = 1.0f;
                if constexpr (!BF) {
                    float m = 0.0f;
                    for (unsigned st = 0; st < steps; st++) {
                        const auto v = part(T::STEP * st + 8 * g);
#pragma unroll
                        for (int i = 0; i < 4; i++) m = fmaxf(m, fmaxf(fabsf(v.a[i]), fabsf(v.b[i])));
                    }
                    const unsigned e = max(__float_as_uint(T::most(m)) >> 23, 15u);
                    up = __uint_as_float((268u - e) << 23);
                    down = __uint_as_float((e - 14u) << 23);
                }
                for (unsigned st = 0; st < steps; st++) {
                    const unsigned j = T::STEP * st + 8 * g;
                    const auto v = part(j);
                    float x[8];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        x[i] = v.a[i] * up;
                        x[4 + i] = v.b[i] * up;
                    }
                    u32x4 w[NRT];
#pragma unroll
                    for (int rt = 0; rt < NRT; rt++) {
                        const unsigned o = o0 + M * rt + col;
                        w[rt] = u32x4{0, 0, 0, 0};
                        if (o >= first && o < end && j < l.rank) w[rt] = ldg<u32x4>(b + (uint64_t)o * l.rank + j);
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
                            const bf16x8 wb = __builtin_bit_cast(bf16x8, w[rt]);
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
                            const f16x8 wh = __builtin_bit_cast(f16x8, w[rt]);
                            d[rt] = T::mfma(wh, p1, d[rt]);
                            d[rt] = T::mfma(wh, p0, d[rt]);
                        }
                    }
                }
                const float f = down * alpha;
#pragma unroll
                for (int rt = 0; rt < NRT; rt++) {
#pragma unroll
                    for (int i = 0; i < N; i++)
                        if (mine) add(rt, i, d[rt][i] * f);
                }
            }
            first = end;
        }
    }
}

// The description checked and brought into the kernels' form; `what` names the call.
int lora_check(const char* what, const g4_lora* l);
LoraDev lora_dev(const g4_lora* l, uint32_t n_tokens);
// Pieces of k that the down product takes, the bytes of its sums, and those that serve every call of no more tokens.
uint32_t lora_splits(const g4_lora* l, uint32_t n_tokens);
size_t lora_bytes(const g4_lora* l, uint32_t n_tokens);
size_t lora_most_bytes(const g4_lora* l, uint32_t n_tokens);
// The down product of every token that has an adapter; d.u and d.ids set. x: rows of x_type, x_scales with e4m3.
void lora_launch_down(const LoraDev& d, uint32_t lora_type, const void* x, uint32_t x_type, uint64_t x_stride,
                      const float* x_scales, hipStream_t st);

}  // namespace g4
