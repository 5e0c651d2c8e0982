// Projections of a served batch in 8 bits (g4_linear_e4m3):
//   out[t][o] = x_scales[t] * weight_scales[o] * sum_k x[t][k] weight[o][k]
// and, in the same launch's epilogue, the requests' low-rank adapters (lora.h).
//
// The 8-bit MFMA adds products eight at a time (k 8 i to 8 i + 7), each cut off below 2^-13 of the power of two of the
// largest of its eight (subnormal codes counted as 2^-6, zeros not at all); the eights' sums are added in f32 (probed product
// by product, and held to it by the tests).
// Elements widened to f16, which is exact, give sums in f32 on the f16 unit, at half the 8-bit unit's rate. f32 outputs
// take that, and 16-bit ones where the caller asks for it (G4_F32_SUMS). Else f16 and bf16 outputs take the 8-bit unit in
// the staged form (and the f16 unit in the form for few tokens, which waits for memory): the root mean square of its error
// is 0.08 of that of f16's own rounding for normal rows, 0.14 with channels 20 times the others, 0.3 with channels 100
// times (at n 1536 and at 8192; bf16's rounding is 8 times f16's). Where large products cancel, what is left has their
// absolute error. Weight rows are the matrix operand's rows, tokens its columns: a lane ends with four consecutive
// outputs of one token.
//
// Measured (us; the library's 8-bit product of the same shape beside): 8192 by 8192 by 8192 440, 2.5 PFLOP/s (408); 4096 tokens
// by 12288 outputs of 1536 92 (74); 64 tokens by the same 7.6 (the weights' bytes at a copy's rate: 4); one token by 2560
// outputs of 1536 3.5. Sums in f32 for 16-bit outputs, without and with: 426 / 792, 85 / 135 and 7.8 / 10.9.
#include <utility>

#include "launch_rules.h"
#include "lora.h"

namespace g4 {

struct Linear8Args {
    const uint8_t* __restrict__ x;
    const uint8_t* __restrict__ w;
    const float* __restrict__ x_scales;
    const float* __restrict__ w_scales;
    void* __restrict__ out;
    uint64_t x_stride, out_stride;
    uint32_t n_tokens, rows, n;
    uint32_t out_type, low;  // low: 0 no adapters, else their type
    uint32_t wide;           // sums in f32 whatever the outputs' type
    LoraDev l;
};

// 32 bytes of a row at k, those past n as 0 (n a multiple of 16).
struct Row32 {
    u32x4 v[2];
};
__device__ __forceinline__ Row32 row32(const uint8_t* p, unsigned k, unsigned n) {
    Row32 r = {{{0, 0, 0, 0}, {0, 0, 0, 0}}};
    if (k < n) r.v[0] = ldg<u32x4>(p + k);
    if (k + 16 < n) r.v[1] = ldg<u32x4>(p + k + 16);
    return r;
}
// Eight e4m3 as f16, exactly.
__device__ __forceinline__ f16x8 widen8(uint32_t a, uint32_t b) {
    f16x8 h;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const uint32_t w = i ? b : a;
        const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false), hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true);
        h[4 * i] = lo[0];
        h[4 * i + 1] = lo[1];
        h[4 * i + 2] = hi[0];
        h[4 * i + 3] = hi[1];
    }
    return h;
}

__device__ __forceinline__ f16x8 widen8(const Row32& r, int q) {  // the q-th eight of 32
    return widen8(r.v[q / 2][2 * (q & 1)], r.v[q / 2][2 * (q & 1) + 1]);
}

// The scales of a 16-output tile's element of the lane's.
struct TileScales {
    float x;
    f32x4 w;
};
__device__ __forceinline__ TileScales tile_scales(const Linear8Args& a, unsigned o0, unsigned t) {
    const unsigned o = o0 + 4 * ((threadIdx.x & 63) >> 4);
    TileScales s;
    s.x = a.x_scales[min(t, a.n_tokens - 1)];
#pragma unroll
    for (int i = 0; i < 4; i++) s.w[i] = a.w_scales[min(o + i, a.rows - 1)];
    return s;
}
// Its sums scaled, the adapters' part added, and stored.
__device__ __forceinline__ void finish(const Linear8Args& a, f32x4 sum, const TileScales& s, unsigned o0, unsigned t) {
    const unsigned o = o0 + 4 * ((threadIdx.x & 63) >> 4);
    const bool valid = t < a.n_tokens;
    f32x4 y;
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = sum[i] * s.x * s.w[i];
    if (a.low) {
        const int id = lora_id(a.l, t, valid);
        auto add = [&](int, int i, float v) __attribute__((always_inline)) { y[i] += v; };
        if (a.low == G4_F16) lora_up<16, 1, false>(a.l, o0, t, id, add);
        else lora_up<16, 1, true>(a.l, o0, t, id, add);
    }
    if (valid && o < a.rows) store4(a.out, a.out_type, t * a.out_stride + o, y, a.rows - o);
}

// Few tokens: 16 RT outputs by 16 CT tokens a workgroup, its waves take every Wth 128 of k.
template <int RT, int CT, int W>
__global__ __launch_bounds__(W * 64) void k_linear8_few(const Linear8Args a) {
    __shared__ f32x4 s_sum[W][RT * CT][64];
    const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
    const unsigned o_tiles = (a.rows + 16 * RT - 1) / (16 * RT), o0 = blockIdx.x % o_tiles * (16 * RT), t0 = blockIdx.x / o_tiles * (16 * CT);
    f32x4 acc[RT][CT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++)
#pragma unroll
        for (int ct = 0; ct < CT; ct++) acc[rt][ct] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const uint8_t *wp[RT], *xp[CT];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) wp[rt] = a.w + (uint64_t)min(o0 + 16 * rt + col, a.rows - 1) * a.n;
#pragma unroll
    for (int ct = 0; ct < CT; ct++) xp[ct] = a.x + min(t0 + 16 * ct + col, a.n_tokens - 1) * a.x_stride;
    struct Operands {
        Row32 w[RT], x[CT];
    };
    auto fetch = [&](unsigned k) __attribute__((always_inline)) {
        Operands r;
#pragma unroll
        for (int rt = 0; rt < RT; rt++) r.w[rt] = row32(wp[rt], k, a.n);
#pragma unroll
        for (int ct = 0; ct < CT; ct++) r.x[ct] = row32(xp[ct], k, a.n);
        return r;
    };
    // The end's scales come with the first operands.
    const unsigned first = wave < RT * CT ? wave : 0;
    const TileScales scales = tile_scales(a, o0 + 16 * (first / CT), t0 + 16 * (first % CT) + col);
    for (unsigned k0 = wave * 128; k0 < a.n; k0 += W * 128) {
        const Operands now = fetch(k0 + 32 * g);
#pragma unroll
        for (int q = 0; q < 4; q++) {
            f16x8 wh[RT];
#pragma unroll
            for (int rt = 0; rt < RT; rt++) wh[rt] = widen8(now.w[rt], q);
#pragma unroll
            for (int ct = 0; ct < CT; ct++) {
                const f16x8 xh = widen8(now.x[ct], q);
#pragma unroll
                for (int rt = 0; rt < RT; rt++) acc[rt][ct] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wh[rt], xh, acc[rt][ct], 0, 0, 0);
            }
        }
    }
#pragma unroll
    for (int rt = 0; rt < RT; rt++)
#pragma unroll
        for (int ct = 0; ct < CT; ct++) s_sum[wave][rt * CT + ct][lane] = acc[rt][ct];
    __syncthreads();
    for (unsigned i = wave; i < RT * CT; i += W) {
        f32x4 s = s_sum[0][i][lane];
#pragma unroll
        for (int w = 1; w < W; w++) s += s_sum[w][i][lane];
        const unsigned o = o0 + 16 * (i / CT), t = t0 + 16 * (i % CT) + col;
        finish(a, s, i == wave ? scales : tile_scales(a, o, t), o, t);
    }
}

// ---- many tokens ---------------------------------------------------------------------
//
// 64 RT outputs by 64 CT tokens a workgroup of four waves, two by two, a wave 2 RT x 2 CT / 4 tiles of 32 x 32. Both
// operands come to LDS by DMA, 64 k a stage, four stages; a wave reads the next stage's operands into registers
// while it multiplies this one's, so LDS, the DMA and the matrix unit work at once, with one barrier a stage. The
// workgroup goes on to its next tile without a pause: the DMA runs up to four stages ahead, across the tiles' ends.
//
// What bounds it: at 8192 cubed the matrix unit is busy 0.73 of the cycles, and the chip runs them at 1.6 GHz: with
// neither DMA nor LDS reads the same products take 0.61 of the time, at 2.2 GHz. Four waves of 128 by 128 (a third fewer LDS
// reads, one wave a SIMD) took 5 % longer: nothing covers a wave's own requests. Tiles of 256 by 128, two workgroups a
// CU, 24 % longer. A tile's stores go on under the next tile's first stages; through LDS, as whole lines, they took longer
// (12288 outputs: 98 against 92 us), as they wait for each other's patches.
//
// A stage holds 64 bytes a row, 16-byte piece c of row r at r * 64 + (c ^ (r / 4) % 4) * 16: sixteen lanes that read one
// piece of sixteen rows meet all 64 banks.
constexpr unsigned kStageK = 64;
// All but the N newest requests have come, the wave's LDS reads too; then every wave's.
template <int N>
__device__ __forceinline__ void stage_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

struct TileArgs {
    Linear8Args a;
    uint32_t o_tiles, t_tiles;
};

// Tiles in an order that keeps the 32 workgroups of an XCD (workgroup b: XCD b % 8) on few rows of both operands at a
// time: each XCD has a run of the order, in which eight token tiles go together.
__device__ __forceinline__ uint32_t tile_begin(uint32_t n, uint32_t part) { return n / 8 * part + min(part, n % 8); }
__device__ __forceinline__ uint2 tile_place(uint32_t i, uint32_t o_tiles, uint32_t t_tiles) {  // x: outputs', y: tokens'
    const uint32_t group = i / (8 * o_tiles), r = i - group * 8 * o_tiles, wide = min(8u, t_tiles - group * 8), o = r / wide;
    return make_uint2(o, group * 8 + r - o * wide);
}

// f(0), f(1) .. f(N - 1), the numbers as types: what depends on them is settled when it is compiled.
template <int... I, typename F>
__device__ __forceinline__ void each_of(std::integer_sequence<int, I...>, F&& f) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void each_of(F&& f) {
    each_of(std::make_integer_sequence<int, N>{}, f);
}

// OT: the outputs' type; kWide16: either 16-bit type, known at run time, and sums in f32. LOW: the adapters' type, 0 none.
constexpr uint32_t kWide16 = 16;
template <int WO, int WT, int RT, int CT, int kStages, uint32_t OT, uint32_t LOW>
__global__ __launch_bounds__(64 * WO * WT, RT * CT >= 16 ? 1 : 2) void k_linear8_tiles(const TileArgs ta) {
    constexpr bool WIDE = OT == G4_F32 || OT == kWide16;
    constexpr int W = WO * WT, OPS = RT + CT, READS = 2 * OPS, PAIRS = RT * CT;
    constexpr unsigned BO = 32 * WO * RT, BT = 32 * WT * CT, STAGE = (BO + BT) * kStageK;
    constexpr int DW = BO / 16 / W, DX = BT / 16 / W, DMAS = DW + DX;  // requests a wave and stage
    static_assert(BO % (16 * W) == 0 && BT % (16 * W) == 0, "even shares");
    constexpr unsigned SLOTS = 4, SCALES = kStages * STAGE;  // scales of up to four tiles: the DMA is two tiles ahead at most
    static_assert(BO % 64 == 0 && BT % 64 == 0, "whole waves of scales");
    __shared__ __attribute__((aligned(16))) uint8_t s_mem[SCALES + SLOTS * (BO + BT) * 4];
    const Linear8Args& a = ta.a;
    const uint32_t type = OT == kWide16 ? a.out_type : OT;
    const unsigned lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned wo = wave / WT * 32 * RT, wt = wave % WT * 32 * CT;
    const uint32_t lds = (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)s_mem);
    const uint32_t tiles = ta.o_tiles * ta.t_tiles, xcd = blockIdx.x % 8;
    const bool even = gridDim.x % 8 == 0;
    const uint32_t tile_0 = even ? tile_begin(tiles, xcd) + blockIdx.x / 8 : blockIdx.x;
    const uint32_t tile_end = even ? tile_begin(tiles, xcd + 1) : tiles, tile_step = even ? gridDim.x / 8 : gridDim.x;
    if (tile_0 >= tile_end) return;
    const unsigned stages = ((a.n + 2 * kStageK - 1) / (2 * kStageK)) * 2;  // of a tile; even

    // The DMA's side: pieces of 16 rows, DW of the weights' and DX of the tokens' a wave; a lane's offset from the tile.
    const char *d_w, *d_x;  // the tile's rows at the stage's k
    uint32_t from[DMAS];
    unsigned d_k = 0, d_tile = tile_0, d_slot = 0;
    uint32_t d_lds = 0;
    auto aim = [&]() __attribute__((always_inline)) {
        const uint2 at = tile_place(d_tile, ta.o_tiles, ta.t_tiles);
        const unsigned o = at.x, t = at.y;
        unsigned l = lane;
        asm volatile("" : "+v"(l));
        const unsigned piece = ((l & 3) ^ ((l >> 4) & 3)) * 16;
        d_w = uniform_ptr(reinterpret_cast<const char*>(a.w) + (uint64_t)(o * BO) * a.n);
        d_x = uniform_ptr(reinterpret_cast<const char*>(a.x) + (uint64_t)(t * BT) * a.x_stride);
#pragma unroll
        for (int j = 0; j < DMAS; j++) {
            const unsigned r = 16 * (j < DW ? wave * DW + j : wave * DX + j - DW) + (l >> 2);
            from[j] = (j < DW ? min(r, a.rows - 1 - o * BO) * a.n : min(r, a.n_tokens - 1 - t * BT) * (uint32_t)a.x_stride) + piece;
        }
#pragma unroll
        for (unsigned first = wave * 64; first < BO + BT; first += 64 * W) {  // 64 of the weights' or of the tokens'
            const unsigned i = first + l;
            scale_dma(first < BO ? a.w_scales + min(o * BO + i, a.rows - 1) : a.x_scales + min(t * BT + i - BO, a.n_tokens - 1),
                      __builtin_amdgcn_readfirstlane(lds + SCALES + (d_slot * (BO + BT) + first) * 4));
        }
        d_slot = (d_slot + 1) % SLOTS;
    };
    auto request = [&](auto j) __attribute__((always_inline)) {
        constexpr unsigned at = j < DW ? j * 1024 : BO * kStageK + (j - DW) * 1024;
        const char* base = j < DW ? d_w : d_x;
        const uint32_t to = lds + d_lds + wave * (j < DW ? DW : DX) * 1024;
        if (d_k + kStageK <= a.n) {  // uniform
            stage_dma<at>(base, from[j], to);
        } else {
            const char* p = base + from[j];
            unsigned l = lane;
            asm volatile("" : "+v"(l));
            if (d_k + ((l & 3) ^ ((l >> 4) & 3)) * 16 >= a.n) p = reinterpret_cast<const char*>(kZeros);
            stage_dma<at>(p, to);
        }
    };
    auto requested = [&]() __attribute__((always_inline)) {  // a stage's; past the last tile the same tile's come again
        d_lds = d_lds == (kStages - 1) * STAGE ? 0 : d_lds + STAGE;
        d_k += kStageK;
        d_w = uniform_ptr(d_w + kStageK);
        d_x = uniform_ptr(d_x + kStageK);
        if (d_k == stages * kStageK) {
            d_k = 0;
            if (d_tile + tile_step < tile_end) d_tile += tile_step;
            aim();
        }
    };
    aim();
#pragma unroll 1
    for (int s = 0; s < kStages; s++) {
        each_of<DMAS>(request);
        requested();
    }

    // The matrix unit's side.
    unsigned off0, off1;  // of the lane's two pieces of a row
    auto place = [&]() __attribute__((always_inline)) {
        unsigned l = lane;
        asm volatile("" : "+v"(l));
        const unsigned col = l & 31, g = l >> 5, swz = (col >> 2) & 3;
        off0 = col * kStageK + ((2 * g) ^ swz) * 16;
        off1 = col * kStageK + ((2 * g + 1) ^ swz) * 16;
    };
    place();
    i32x8 reg[2][OPS];
    unsigned r_lds = 0;
    auto read = [&](i32x8 (&to)[OPS], auto i) __attribute__((always_inline)) {
        constexpr int j = i / 2, h = i % 2;
        const unsigned base = r_lds + (j < RT ? wo * kStageK + j * 32 * kStageK : (BO + wt) * kStageK + (j - RT) * 32 * kStageK);
        const u32x4 v = *reinterpret_cast<const u32x4*>(s_mem + base + (h ? off1 : off0));
#pragma unroll
        for (int e = 0; e < 4; e++) to[j][4 * h + e] = (int)v[e];
    };
    stage_barrier<(kStages - 1) * DMAS>();
    each_of<READS>([&](auto i) __attribute__((always_inline)) { read(reg[0], i); });
    r_lds = STAGE;
    stage_barrier<(kStages - 2) * DMAS>();

    f32x16 acc[RT][CT];
    bool stored = false;  // whether the tile before left PAIRS * (4 or 2) stores, all of them
    unsigned slot = 0;
    auto stage = [&](const i32x8 (&now)[OPS], i32x8 (&next)[OPS], auto first, auto early) __attribute__((always_inline)) {
        constexpr int SUBS = WIDE ? 4 : 1, STEPS = PAIRS * SUBS;
        f16x8 half[2][OPS];
        auto widen = [&](auto j, auto q) __attribute__((always_inline)) { half[q & 1][j] = widen8(now[j][2 * q], now[j][2 * q + 1]); };
        if constexpr (WIDE) each_of<OPS>([&](auto j) __attribute__((always_inline)) { widen(j, std::integral_constant<int, 0>{}); });
        each_of<STEPS>([&](auto m) __attribute__((always_inline)) {
            constexpr int q = m / PAIRS, pair = m % PAIRS, rt = pair / CT, ct = rt & 1 ? CT - 1 - pair % CT : pair % CT;
            f32x16 c = acc[rt][ct];
            if constexpr (first && q == 0) c = f32x16{0};
            if constexpr (WIDE) acc[rt][ct] = __builtin_amdgcn_mfma_f32_32x32x16_f16(half[q & 1][rt], half[q & 1][RT + ct], c, 0, 0, 0);
            else acc[rt][ct] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(now[rt], now[RT + ct], c, 0, 0, 0, 0, 0, 0);
            if constexpr (WIDE && q < 3) {
                // The next quarter's elements, evenly over this one's products.
                constexpr int w0 = pair * OPS / PAIRS, w1 = (pair + 1) * OPS / PAIRS;
                each_of<w1 - w0>([&](auto j) __attribute__((always_inline)) {
                    widen(std::integral_constant<int, w0 + j>{}, std::integral_constant<int, q + 1>{});
                });
            }
            // The reads in the first part, the DMA's requests all along.
            constexpr int by = STEPS > 1 ? STEPS * 3 / 4 : 1;
            constexpr int r0 = m < by ? m * READS / by : READS, r1 = m + 1 < by ? (m + 1) * READS / by : READS;
            each_of<r1 - r0>([&](auto i) __attribute__((always_inline)) { read(next, std::integral_constant<int, r0 + i>{}); });
            constexpr int d0 = m * DMAS / STEPS, d1 = (m + 1) * DMAS / STEPS;
            each_of<d1 - d0>([&](auto j) __attribute__((always_inline)) { request(std::integral_constant<int, d0 + j>{}); });
            __builtin_amdgcn_sched_barrier(0);
        });
        requested();
        r_lds = r_lds == (kStages - 1) * STAGE ? 0 : r_lds + STAGE;
        // The last tile's stores are younger than the stages that the first two barriers wait for: they may go on.
        constexpr int AFTER = (kStages - 2) * DMAS + PAIRS * (OT == G4_F32 ? 4 : 2);  // the counter's most is 63
        if (decltype(early)::value && stored) stage_barrier<AFTER < 63 ? AFTER : 63>();
        else stage_barrier<(kStages - 2) * DMAS>();
    };
    constexpr std::true_type kFirst{};  // of a tile: nothing to add to; the tile before may have left stores
    constexpr std::false_type kLater{};

    for (unsigned i = tile_0; i < tile_end; i += tile_step) {
        stage(reg[0], reg[1], kFirst, kFirst);
        stage(reg[1], reg[0], kLater, kFirst);
#pragma unroll 1
        for (unsigned s = 2; s < stages; s += 2) {
            stage(reg[0], reg[1], kLater, kLater);
            stage(reg[1], reg[0], kLater, kLater);
        }
        const uint2 at = tile_place(i, ta.o_tiles, ta.t_tiles);
        const unsigned o0 = at.x * BO + wo, t0 = at.y * BT + wt;
        unsigned el = lane;  // what follows from it is not kept beside the next tile's sums
        asm volatile("" : "+v"(el));
        const unsigned col = el & 31, g = el >> 5;
        const float* scales = reinterpret_cast<const float*>(s_mem + SCALES) + slot * (BO + BT);
        slot = (slot + 1) % SLOTS;
        stored = o0 + 32 * RT <= a.rows && t0 + 32 * CT <= a.n_tokens;  // uniform: every lane stores whole pieces
        each_of<CT>([&](auto ct) __attribute__((always_inline)) {
            const unsigned t = t0 + 32 * ct + col;
            const float xs = scales[BO + wt + 32 * ct + col];
            const int id = LOW ? lora_id(a.l, t, t < a.n_tokens) : -1;
            constexpr int TOGETHER = LOW != 0 && PAIRS < 8 ? RT : 1;  // row tiles that share the adapters' sums of a token
            f32x4 y[TOGETHER][4];
            each_of<RT>([&](auto rt) __attribute__((always_inline)) {
                const unsigned o = o0 + 32 * rt;
                if constexpr (rt % TOGETHER == 0) {
                    each_of<TOGETHER>([&](auto r) __attribute__((always_inline)) {
                        each_of<4>([&](auto q) __attribute__((always_inline)) {
                            const f32x4 ws = *reinterpret_cast<const f32x4*>(scales + wo + 32 * (rt + r) + 8 * q + 4 * g);
#pragma unroll
                            for (int e = 0; e < 4; e++) y[r][q][e] = acc[rt + r][ct][4 * q + e] * xs * ws[e];
                        });
                    });
                    if constexpr (LOW != 0) {
                        auto add = [&](int r, int i, float v) __attribute__((always_inline)) { y[r][i / 4][i % 4] += v; };
                        lora_up<32, TOGETHER, LOW == G4_BF16, (PAIRS < 8)>(a.l, o, t, id, add);
                    }
                }
                const f32x4(&yr)[4] = y[rt % TOGETHER];
                if (!stored) {
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const unsigned oq = o + 8 * q + 4 * g;
                        if (t < a.n_tokens && oq < a.rows)
                            store4(a.out, type, t * a.out_stride + oq, yr[q], a.rows - oq);
                    }
                } else if constexpr (OT == G4_F32) {
                    float* out = static_cast<float*>(a.out) + t * a.out_stride + o + 4 * g;
#pragma unroll
                    for (int q = 0; q < 4; q++) *(__attribute__((address_space(1))) f32x4_any*)(out + 8 * q) = yr[q];
                } else {
                    // Lane halves exchange, so that a lane has eight outputs one after the other: the lower half's of every
                    // even eight, the upper's of the odd.
                    uint16_t* out = static_cast<uint16_t*>(a.out) + t * a.out_stride + o + 8 * g;
#pragma unroll
                    for (int q = 0; q < 4; q += 2) {
                        uint32_t w[2][2];
#pragma unroll
                        for (int p = 0; p < 2; p++)
#pragma unroll
                            for (int e = 0; e < 2; e++) w[p][e] = pair16(yr[q + p][2 * e], yr[q + p][2 * e + 1], type);
                        u32x4 v;
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const auto sw = __builtin_amdgcn_permlane32_swap(w[0][e], w[1][e], false, false);
                            v[e] = sw[0];
                            v[2 + e] = sw[1];
                        }
                        *(__attribute__((address_space(1))) u32x4_any*)(out + 8 * q) = v;
                    }
                }
                __builtin_amdgcn_sched_barrier(0);  // tile by tile: the registers hold no more
            });
        });
        if (!stored) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // an unknown number of stores: the counts begin anew
        if constexpr (LOW != 0) {  // the next tile's first operands once more: the adapters need the registers in between
            asm volatile("" ::: "memory");
            place();
            const unsigned ahead = r_lds;
            r_lds = ahead == 0 ? (kStages - 1) * STAGE : ahead - STAGE;
            each_of<READS>([&](auto j) __attribute__((always_inline)) { read(reg[0], j); });
            r_lds = ahead;
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the next stage's requests go where these lay
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no DMA into LDS that is another workgroup's by then
}

}  // namespace g4

using namespace g4;

namespace {

int linear8_check(const g4_linear_e4m3_params* p, const g4_lora* lora) {
    const char* what = "linearE4m3";
    if (!p) return fail(G4_EINVAL, "%s: NULL params", what);
    if (p->n_tokens > kMaxRows) return fail(G4_EINVAL, "%s: %u tokens (at most 2^22)", what, p->n_tokens);
    if (p->rows == 0 || p->rows > (1u << 20)) return fail(G4_EINVAL, "%s: %u rows (1 to 2^20)", what, p->rows);
    if (p->n == 0 || p->n % 16 || p->n > 65536) return fail(G4_EINVAL, "%s: n %u (a multiple of 16, at most 65536)", what, p->n);
    if ((p->out_type & ~G4_F32_SUMS) > G4_BF16) return fail(G4_EINVAL, "%s: out_type %u (f32, f16 or bf16)", what, p->out_type);
    if (p->x_stride && p->x_stride < p->n) return fail(G4_EINVAL, "%s: x_stride below n %u", what, p->n);
    if (p->out_stride && p->out_stride < p->rows) return fail(G4_EINVAL, "%s: out_stride below the rows %u", what, p->rows);
    if (p->x_stride > (1ull << 40) || p->out_stride > (1ull << 40)) return fail(G4_EINVAL, "%s: a stride is too long", what);
    if (!lora) return G4_OK;
    const int rc = lora_check(what, lora);
    if (rc) return rc;
    uint32_t rows = 0;
    for (uint32_t s = 0; s < lora->n_segs; s++) rows += lora->widths[s];
    if (lora->n != p->n || rows != p->rows)
        return fail(G4_EINVAL, "%s: adapters of %u inputs and %u outputs beside a projection of %u and %u", what, lora->n, rows, p->n,
                    p->rows);
    return G4_OK;
}

template <int WO, int WT, int RT, int CT, int NS>
void launch_tiles(const Linear8Args& a, hipStream_t st) {
    constexpr uint32_t BO = 32 * WO * RT, BT = 32 * WT * CT;
    TileArgs t = {a, (a.rows + BO - 1) / BO, (a.n_tokens + BT - 1) / BT};
    const uint32_t n = t.o_tiles * t.t_tiles, most = device_cus() * (BO * BT >= 65536 ? 1 : BO * BT >= 16384 ? 2 : 4);
    const dim3 grid(n < most ? n : most), block(64 * WO * WT);
    auto launch = [&](auto type) {
        constexpr uint32_t OT = decltype(type)::value;
        if (a.low == G4_F16) G4_LAUNCH((k_linear8_tiles<WO, WT, RT, CT, NS, OT, G4_F16>), grid, block, 0, st, t);
        else if (a.low) G4_LAUNCH((k_linear8_tiles<WO, WT, RT, CT, NS, OT, G4_BF16>), grid, block, 0, st, t);
        else G4_LAUNCH((k_linear8_tiles<WO, WT, RT, CT, NS, OT, 0>), grid, block, 0, st, t);
    };
    if (a.out_type == G4_F32) launch(std::integral_constant<uint32_t, G4_F32>{});
    else if (a.wide) launch(std::integral_constant<uint32_t, kWide16>{});
    else if (a.out_type == G4_F16) launch(std::integral_constant<uint32_t, G4_F16>{});
    else launch(std::integral_constant<uint32_t, G4_BF16>{});
}

template <int RT, int CT, int W>
void launch_few(const Linear8Args& a, hipStream_t st) {
    const uint32_t o_tiles = (a.rows + 16 * RT - 1) / (16 * RT), t_tiles = (a.n_tokens + 16 * CT - 1) / (16 * CT);
    G4_LAUNCH((k_linear8_few<RT, CT, W>), dim3(o_tiles * t_tiles), dim3(W * 64), 0, st, a);
}

// Tiles by the rule; else tiles of 16 or 32 whose waves share k: 16 outputs by 16 tokens (us, n 1536: one token by 2560 3.5, 32
// outputs 4.3), 32 by 32 up to 96 tokens (64 by 2560 5.7, 32 by 64 7.2), above 32 by 64 (128 by 2560 7.6, 8.5).
void launch_linear8(const Linear8Args& a, hipStream_t st) {
    const uint32_t side = linear8_tile(a.n_tokens, a.rows, a.x_stride, device_cus());
    if (side == 256) launch_tiles<2, 4, 4, 2, 4>(a, st);
    else if (side == 128) launch_tiles<2, 2, 2, 2, 4>(a, st);
    else if (side == 64) launch_tiles<2, 2, 1, 1, 4>(a, st);
    else if (a.n_tokens <= 16) launch_few<1, 1, 8>(a, st);
    else if (a.n_tokens <= 96) launch_few<2, 2, 8>(a, st);
    else launch_few<2, 4, 8>(a, st);
}

}  // namespace

extern "C" {

int g4_linear_e4m3_workspace_size(const g4_linear_e4m3_params* p, const g4_lora* lora, size_t* bytes) {
    if (!bytes) return fail(G4_EINVAL, "g4_linear_e4m3_workspace_size: bytes is NULL");
    const int rc = linear8_check(p, lora);
    if (rc) return rc;
    *bytes = 16 + (lora ? lora_bytes(lora, p->n_tokens) : 0);
    return G4_OK;
}

int g4_linear_e4m3(const uint8_t* x, const float* x_scales, const uint8_t* weight, const float* weight_scales,
                   const g4_lora* lora, const int32_t* adapter_ids, void* out, const g4_linear_e4m3_params* p, void* workspace,
                   size_t workspace_bytes, void* stream) {
    const char* what = "linearE4m3";
    const int rc = linear8_check(p, lora);
    if (rc) return rc;
    if (!x || !x_scales || !weight || !weight_scales || !out || !workspace)
        return fail(G4_EINVAL, "%s: NULL x, weight, scales, out or workspace", what);
    if (!lora != !adapter_ids) return fail(G4_EINVAL, "%s: lora and adapter_ids go together", what);
    const uint64_t xs = p->x_stride ? p->x_stride : p->n, os = p->out_stride ? p->out_stride : p->rows;
    if (!aligned(x, 16) || !aligned(weight, 16) || xs % 16) return fail(G4_EINVAL, "%s: rows must be 16-byte aligned", what);
    const uint32_t out_type = p->out_type & ~G4_F32_SUMS, width = type_bytes(out_type);
    if (!aligned(x_scales, 4) || !aligned(weight_scales, 4) || !aligned(adapter_ids, 4) || !aligned(out, width))
        return fail(G4_EINVAL, "%s: misaligned scales, adapter_ids or out", what);
    if (!aligned(workspace, 16)) return fail(G4_EINVAL, "%s: workspace must be 16-byte aligned", what);
    const size_t low = lora ? lora_bytes(lora, p->n_tokens) : 0;
    if (workspace_bytes < low) return fail(G4_ENOSPC, "%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, low);
    if (p->n_tokens == 0) return G4_OK;
    Linear8Args a = {};
    a.x = x;
    a.w = weight;
    a.x_scales = x_scales;
    a.w_scales = weight_scales;
    a.out = out;
    a.x_stride = xs;
    a.out_stride = os;
    a.n_tokens = p->n_tokens;
    a.rows = p->rows;
    a.n = p->n;
    a.out_type = out_type;
    a.wide = (p->out_type & G4_F32_SUMS) != 0;
    const hipStream_t st = as_stream(stream);
    const Operand o_x = rows_operand("x", x, G4_E4M3, p->n, xs, p->n_tokens), o_xs = {"x_scales", one_range(x_scales, 4ull * p->n_tokens)},
                  o_w = {"weight", one_range(weight, (uint64_t)p->rows * p->n)},
                  o_ws = {"weight_scales", one_range(weight_scales, 4ull * p->rows)},
                  o_out = rows_operand("out", out, out_type, p->rows, os, p->n_tokens);
    int meet = apart_check(what, o_out, {o_x, o_xs, o_w, o_ws});
    if (meet) return meet;
    if (lora) {
        a.low = lora->type;
        a.l = lora_dev(lora, p->n_tokens);
        a.l.ids = adapter_ids;
        a.l.u = static_cast<float*>(workspace);
        const LoraOperands l = lora_operands(a.l);  // a, the down rows, are read before out is written
        meet = apart_check(what, l.u, {o_x, o_xs, o_w, o_ws, l.a, l.b, l.scales, l.ids, o_out});
        if (!meet) meet = apart_check(what, o_out, {l.b, l.scales, l.ids});
        if (meet) return meet;
        lora_launch_down(a.l, lora->type, x, G4_E4M3, xs, x_scales, st);
        G4_CHECK_LAUNCH("k_lora_down");
    }
    launch_linear8(a, st);
    G4_CHECK_LAUNCH("k_linear8");
    return G4_OK;
}

}  // extern "C"
