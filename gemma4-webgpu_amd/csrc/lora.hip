// Low-rank adapters of many requests beside a projection made elsewhere
// (g4_lora_add), and the down product that linear8.hip shares.
//
// Bound by latency for few tokens (one token's q, k, v of rank 16: 2.9 us down, 3.8 up, two launches that each wait for
// ids, rows and sums in turn; 64 requests of 40 adapters beside their projection: 3.4 us down, 8.0 for the projection with
// the up product in it), by the adapters' way through the caches for many: a tile of 16 tokens reads all of
// its adapter (4003 tokens, n 2048, rank 64: 9.5 us for 64 MB of them).
#include <type_traits>

#include "lora.h"

namespace g4 {

// How x and the adapters' rows meet. 16-bit products are exact in f32, and so is an e4m3 element as f16 or bf16; f32 rows,
// and 16-bit ones of the adapters' other type (mixed), meet them as f32.
enum { kDownF16, kDownBf16, kDownE4m3F16, kDownE4m3Bf16, kDownF32, kDownMixed };

struct DownArgs {
    LoraDev l;
    const void* __restrict__ x;
    const float* __restrict__ x_scales;
    uint64_t x_stride;
    uint32_t x_type, a_type;
};

// 8 e4m3 as f16 or bf16, exactly.
template <bool BF>
__device__ __forceinline__ u32x4 e4m3_wide(u32x2 q) {
    u32x4 r;
#pragma unroll
    for (int w = 0; w < 2; w++) {
        if constexpr (BF) {
            const auto lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[w], 1.0f, false), hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[w], 1.0f, true);
            r[2 * w] = __builtin_bit_cast(uint32_t, lo);
            r[2 * w + 1] = __builtin_bit_cast(uint32_t, hi);
        } else {
            const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(q[w], 1.0f, false), hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(q[w], 1.0f, true);
            r[2 * w] = __builtin_bit_cast(uint32_t, lo);
            r[2 * w + 1] = __builtin_bit_cast(uint32_t, hi);
        }
    }
    return r;
}

// 8 elements of a 16-bit type as f32.
__device__ __forceinline__ void wide8(float (&v)[8], u32x4 q, uint32_t type) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float h = h2f((uint16_t)(q[i / 2] >> (16 * (i & 1)))), b = __uint_as_float((i & 1) ? q[i / 2] & 0xFFFF0000u : q[i / 2] << 16);
        v[i] = type == G4_F16 ? h : b;
    }
}

// Few tokens: a wave takes four down rows of one token, its lanes eight k at a time; no adapter waits for another.
constexpr int kFewRows = 4, kFewWaves = 4;
template <uint32_t XT, bool BF>
__global__ __launch_bounds__(kFewWaves * 64) void k_lora_down_few(const DownArgs a) {
    const LoraDev& l = a.l;
    const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6, t = blockIdx.x;
    const unsigned r0 = (blockIdx.y * kFewWaves + wave) * kFewRows;
    const int id = lora_id(l, t, true);
    if (id < 0 || r0 >= l.down) return;
    const uint16_t* rows = static_cast<const uint16_t*>(l.a) + ((uint64_t)id * l.down + r0) * l.n;  // l.down: a multiple of 4
    const char* x = static_cast<const char*>(a.x) + t * a.x_stride * (XT == G4_F32 ? 4 : XT == G4_E4M3 ? 1 : 2);
    float sum[kFewRows] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 2
    for (unsigned k0 = 0; k0 < l.n; k0 += 512) {
        const unsigned k = k0 + 8 * lane;
        if (k >= l.n) continue;
        u32x4 w[kFewRows];
#pragma unroll
        for (int r = 0; r < kFewRows; r++) w[r] = ldg<u32x4>(rows + (uint64_t)r * l.n + k);
        f32x4 lo, hi;
        if constexpr (XT == G4_F32) {
            lo = ldg<f32x4>(x + 4 * k);
            hi = ldg<f32x4>(x + 4 * k + 16);
        } else if constexpr (XT == G4_E4M3) {
            const u32x2 q = ldg<u32x2>(x + k);
            const auto a0 = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[0], false), a1 = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[0], true);
            const auto b0 = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[1], false), b1 = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[1], true);
            lo = f32x4{a0[0], a0[1], a1[0], a1[1]};
            hi = f32x4{b0[0], b0[1], b1[0], b1[1]};
        } else {
            const u32x4 q = ldg<u32x4>(x + 2 * k);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float e = XT == G4_F16 ? h2f((uint16_t)q[i]) : __uint_as_float(q[i] << 16);
                const float o = XT == G4_F16 ? h2f((uint16_t)(q[i] >> 16)) : __uint_as_float(q[i] & 0xFFFF0000u);
                (i < 2 ? lo : hi)[2 * (i & 1)] = e;
                (i < 2 ? lo : hi)[2 * (i & 1) + 1] = o;
            }
        }
#pragma unroll
        for (int r = 0; r < kFewRows; r++) sum[r] = lora_dot8<BF>(w[r], lo, hi, sum[r]);
    }
#pragma unroll
    for (int r = 0; r < kFewRows; r++) {
#pragma unroll
        for (int m = 1; m < 16; m <<= 1) sum[r] += __shfl_xor(sum[r], m);
        sum[r] = add_xor32(add_xor16(sum[r]));
    }
    if (lane == 0) {
        const float xs = a.x_scales ? a.x_scales[t] : 1.0f;
        stg<f32x4>(l.u + (uint64_t)t * l.down + r0, f32x4{sum[0] * xs, sum[1] * xs, sum[2] * xs, sum[3] * xs});
    }
}

// Many tokens: 16 CT tokens by 16 RT down rows a workgroup; the tile's adapters one after the other.
//
// Each wave takes every Wth 64 k and brings both operands of it to LDS by DMA, one chunk ahead: loaded straight into the matrix
// unit's layout, in which neighbouring lanes lie in different rows, every lane's 16 bytes are an access of their own (4003
// tokens, n 2048, rank 64: 21 us). Piece c (16 bytes) of row r lies at c ^ r / 2 % 4 of its 64 bytes, c ^ r % 8 of its 128,
// c ^ r % 16 of its 256. Products in f32 (f32 rows, mixed types) run at a sixteenth of the 16-bit rate, after the widening: 4003
// tokens, n 2048, rank 64 and the up product to 2560 take 60 us, with equal 16-bit types 45.
constexpr int kDownWaves = 4;
template <int N>
__device__ __forceinline__ void down_wait() {  // all but the N newest requests of the wave
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
template <int MODE, int RT>  // RT tiles of 16 rows
__global__ __launch_bounds__(kDownWaves * 64) void k_lora_down(const DownArgs a) {
    constexpr int CT = 1;  // tiles of 16 tokens
    constexpr bool BF = MODE == kDownBf16 || MODE == kDownE4m3Bf16, E4M3 = MODE == kDownE4m3F16 || MODE == kDownE4m3Bf16;
    constexpr bool FULL = MODE == kDownF32 || MODE == kDownMixed;  // f32 products
    constexpr unsigned XB = E4M3 ? 1 : MODE == kDownF32 ? 4 : 2, XROW = 64 * XB, XPER = 1024 / XROW, XP = XROW / 16;
    constexpr unsigned WBYTES = RT * 16 * 128, CHUNK = WBYTES + CT * 16 * XROW;
    constexpr int DMAS = CHUNK / 1024;
    constexpr unsigned SUMS = RT * CT * 1024;
    constexpr unsigned AREA = 2 * CHUNK;  // a wave's: two chunks, then its sums
    static_assert(AREA >= SUMS, "the sums take the chunks' place");
    __shared__ __attribute__((aligned(16))) uint8_t s_mem[kDownWaves * AREA];
    __shared__ int s_id[64];
    const LoraDev& l = a.l;
    const unsigned lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
    const unsigned t0 = blockIdx.x * (16 * CT), r0 = blockIdx.y * (16 * RT);
    uint8_t* const mine = s_mem + wave * AREA;
    // Lane: token of the tile. One wave's reading for all, so that they agree whatever happens to the array meanwhile.
    if (wave == 0) s_id[lane] = lora_id(l, t0 + lane, lane < 16 * CT && t0 + lane < l.n_tokens);
    __syncthreads();
    const int id = s_id[lane];
    uint64_t left = __ballot(id >= 0);
    const unsigned chunks = (l.n + 63) / 64;
    while (left) {  // uniform over the workgroup
        const int ad = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
        const uint64_t with = __ballot(id == ad);
        left &= ~with;
        f32x4 acc[RT][CT];
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
#pragma unroll
            for (int ct = 0; ct < CT; ct++) acc[rt][ct] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        const uint32_t lds = __builtin_amdgcn_readfirstlane(
            (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)mine));
        const char* from[DMAS];  // at k = 0
        unsigned at[DMAS];       // the lane's first element of a chunk
#pragma unroll
        for (int j = 0; j < DMAS; j++) {
            if (j < RT * 2) {  // eight rows of 128 bytes
                const unsigned r = 8 * j + (lane >> 3), piece = (lane & 7) ^ (r & 7);
                at[j] = piece * 8;
                from[j] = reinterpret_cast<const char*>(static_cast<const uint16_t*>(l.a) +
                                                        ((uint64_t)ad * l.down + min(r0 + r, l.down - 1)) * l.n + at[j]);
            } else {  // XPER rows of XROW bytes
                const unsigned r = XPER * (j - RT * 2) + lane / XP, turn = E4M3 ? (r >> 1) & 3 : r & (XP - 1), piece = (lane % XP) ^ turn;
                at[j] = piece * (16 / XB);
                from[j] = static_cast<const char*>(a.x) + XB * (min(t0 + r, l.n_tokens - 1) * a.x_stride + at[j]);
            }
        }
        // A chunk into half `half` of the wave's; past the end, and lanes past n, zeros.
        auto request = [&](unsigned c, unsigned half) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < DMAS; j++) {
                const char* p = from[j] + (uint64_t)c * (j < RT * 2 ? 128 : XROW);
                if (c * 64 + at[j] >= l.n) p = reinterpret_cast<const char*>(kZeros);
                stage_dma<0>(p, lds + half * CHUNK + j * 1024);
            }
        };
        unsigned half = 0;
        request(wave, 0);
        for (unsigned c = wave; c < chunks; c += kDownWaves, half ^= 1) {
            request(c + kDownWaves, half ^ 1);
            down_wait<DMAS>();
            const uint8_t* w = mine + half * CHUNK;
            const uint8_t* x = w + WBYTES;
            if constexpr (FULL) {
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    float xf[CT][8], wf[RT][8];
#pragma unroll
                    for (int ct = 0; ct < CT; ct++) {
                        const uint8_t* row = x + (16 * ct + col) * XROW;
                        if constexpr (MODE == kDownF32) {
                            const f32x4 lo = *reinterpret_cast<const f32x4*>(row + ((8 * h + 2 * g) ^ col) * 16);
                            const f32x4 hi = *reinterpret_cast<const f32x4*>(row + ((8 * h + 2 * g + 1) ^ col) * 16);
#pragma unroll
                            for (int e = 0; e < 8; e++) xf[ct][e] = e < 4 ? lo[e] : hi[e - 4];
                        } else {
                            wide8(xf[ct], *reinterpret_cast<const u32x4*>(row + ((4 * h + g) ^ (col & 7)) * 16), a.x_type);
                        }
                    }
#pragma unroll
                    for (int rt = 0; rt < RT; rt++)
                        wide8(wf[rt], *reinterpret_cast<const u32x4*>(w + (16 * rt + col) * 128 + ((4 * h + g) ^ (col & 7)) * 16), a.a_type);
#pragma unroll
                    for (int e = 0; e < 8; e++)
#pragma unroll
                        for (int rt = 0; rt < RT; rt++)
#pragma unroll
                            for (int ct = 0; ct < CT; ct++)
                                acc[rt][ct] = __builtin_amdgcn_mfma_f32_16x16x4f32(wf[rt][e], xf[ct][e], acc[rt][ct], 0, 0, 0);
                }
            } else {
                u32x4 wv[RT][2], xv[CT][2];
#pragma unroll
                for (int h = 0; h < 2; h++) {  // k 32 h + 8 g of the chunk
#pragma unroll
                    for (int rt = 0; rt < RT; rt++)
                        wv[rt][h] = *reinterpret_cast<const u32x4*>(w + (16 * rt + col) * 128 + ((4 * h + g) ^ (col & 7)) * 16);
#pragma unroll
                    for (int ct = 0; ct < CT; ct++) {
                        if constexpr (E4M3) {
                            const unsigned piece = (2 * h + (g >> 1)) ^ ((col >> 1) & 3);
                            xv[ct][h] = e4m3_wide<BF>(*reinterpret_cast<const u32x2*>(x + (16 * ct + col) * 64 + piece * 16 + 8 * (g & 1)));
                        } else {
                            xv[ct][h] = *reinterpret_cast<const u32x4*>(x + (16 * ct + col) * 128 + ((4 * h + g) ^ (col & 7)) * 16);
                        }
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int rt = 0; rt < RT; rt++)
#pragma unroll
                        for (int ct = 0; ct < CT; ct++) {
                            if constexpr (BF)
                                acc[rt][ct] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                    __builtin_bit_cast(bf16x8, wv[rt][h]), __builtin_bit_cast(bf16x8, xv[ct][h]), acc[rt][ct], 0, 0, 0);
                            else
                                acc[rt][ct] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                    __builtin_bit_cast(f16x8, wv[rt][h]), __builtin_bit_cast(f16x8, xv[ct][h]), acc[rt][ct], 0, 0, 0);
                        }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read: the next request but one goes here
        }
        down_wait<0>();  // the last, of zeros, has come too: its place is the sums'
        f32x4* sums = reinterpret_cast<f32x4*>(mine);
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
#pragma unroll
            for (int ct = 0; ct < CT; ct++) sums[(rt * CT + ct) * 64 + lane] = acc[rt][ct];
        __syncthreads();
        for (unsigned i = wave; i < RT * CT; i += kDownWaves) {
            const unsigned rt = i / CT, ct = i % CT, t = t0 + 16 * ct + col, row = r0 + 16 * rt + 4 * g;
            f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < kDownWaves; w++) s += reinterpret_cast<const f32x4*>(s_mem + w * AREA)[i * 64 + lane];
            if (((with >> (16 * ct + col)) & 1) && row < l.down) {  // down and row: multiples of 4
                if (a.x_scales) s *= a.x_scales[t];
                stg<f32x4>(l.u + (uint64_t)t * l.down + row, s);
            }
        }
        __syncthreads();
    }
}

// out = base + the adapters' part. A wave: 16 tokens by TILES * 16 outputs.
constexpr int kUpWaves = 4;
struct UpArgs {
    LoraDev l;
    const void* base;  // may be out
    void* out;
    uint64_t base_stride, out_stride;
    uint32_t type;
};
template <int TILES, bool BF>
__global__ __launch_bounds__(kUpWaves * 64) void k_lora_up(const UpArgs a) {
    const LoraDev& l = a.l;
    const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
    const unsigned t = blockIdx.x * 16 + (lane & 15), o0 = (blockIdx.y * kUpWaves + wave) * (16 * TILES);
    if (o0 >= l.rows) return;
    const bool valid = t < l.n_tokens;
    const int id = lora_id(l, t, valid);
    f32x4 acc[TILES];
#pragma unroll
    for (int rt = 0; rt < TILES; rt++) {
        const unsigned o = o0 + 16 * rt + 4 * g;
        acc[rt] = valid && o < l.rows ? load4(a.base, a.type, t * a.base_stride + o, l.rows - o) : f32x4{0, 0, 0, 0};
    }
    lora_up<16, TILES, BF>(l, o0, t, id, [&](int rt, int i, float v) __attribute__((always_inline)) { acc[rt][i] += v; });
#pragma unroll
    for (int rt = 0; rt < TILES; rt++) {
        const unsigned o = o0 + 16 * rt + 4 * g;
        if (valid && o < l.rows) store4(a.out, a.type, t * a.out_stride + o, acc[rt], l.rows - o);
    }
}

int lora_check(const char* what, const g4_lora* l) {
    if (!l) return fail(G4_EINVAL, "%s: NULL lora", what);
    if (!l->a || !l->b) return fail(G4_EINVAL, "%s: NULL adapters", what);
    if (!aligned(l->a, 16) || !aligned(l->b, 16)) return fail(G4_EINVAL, "%s: adapters must be 16-byte aligned", what);
    if (!aligned(l->scales, 4)) return fail(G4_EINVAL, "%s: misaligned adapter scales", what);
    if (l->n_adapters == 0 || l->n_adapters > 65535) return fail(G4_EINVAL, "%s: %u adapters (1 to 65535)", what, l->n_adapters);
    if (l->rank == 0 || l->rank % 8 || l->rank > kLoraMaxRank)
        return fail(G4_EINVAL, "%s: rank %u (a multiple of 8, at most %u)", what, l->rank, kLoraMaxRank);
    if (l->n == 0 || l->n % 16 || l->n > 65536) return fail(G4_EINVAL, "%s: n %u (a multiple of 16, at most 65536)", what, l->n);
    if (l->n_segs == 0 || l->n_segs > 4) return fail(G4_EINVAL, "%s: %u segments (1 to 4)", what, l->n_segs);
    if (l->type != G4_F16 && l->type != G4_BF16) return fail(G4_EINVAL, "%s: adapter type %u (f16 or bf16)", what, l->type);
    if (l->reserved) return fail(G4_EINVAL, "%s: reserved must be 0", what);
    uint64_t rows = 0;
    for (uint32_t s = 0; s < l->n_segs; s++) {
        if (l->widths[s] == 0) return fail(G4_EINVAL, "%s: segment %u has no outputs", what, s);
        rows += l->widths[s];
    }
    if (rows > (1u << 20)) return fail(G4_EINVAL, "%s: %llu outputs (at most 2^20)", what, (unsigned long long)rows);
    return G4_OK;
}

LoraDev lora_dev(const g4_lora* l, uint32_t n_tokens) {
    LoraDev d = {};
    d.a = l->a;
    d.b = l->b;
    d.scales = l->scales;
    d.n_adapters = l->n_adapters;
    d.rank = l->rank;
    d.n = l->n;
    d.n_segs = l->n_segs;
    uint32_t end = 0;
    for (uint32_t s = 0; s < 4; s++) d.ends[s] = end += s < l->n_segs ? l->widths[s] : 0;
    d.rows = end;
    d.down = l->n_segs * l->rank;
    d.n_tokens = n_tokens;
    return d;
}

size_t lora_bytes(const g4_lora* l, uint32_t n_tokens) { return (size_t)n_tokens * l->n_segs * l->rank * 4 + 16; }

// A wave a token and four rows where that reads at most 64 MB of adapters, no adapter waiting for another; beyond, the
// matrix units' tiles, which read an adapter once for 16 tokens (us of lora_add, 2560 outputs, waves / tiles, f16 and then f32
// rows; four runs of tokens: 256 tokens, rank 64, n 1536 9.6 / 8.3, 9.8 / 10.7; 1024, 16, 1536 13.4 / 12.3, 14.1 / 14.7; 512, 64, 1536
// 13.4 / 10.4, 14.1 / 13.0; 1024, 64, 1536 22.7 / 15.7, 24.4 / 18.1; every token another of 40 adapters, rank 16: 64 tokens 6.6 /
// 26, 6.7 / 66; 1024 27 / 49, 28 / 86). Ids are the device's: what runs of tokens lose here is what mixed ones would lose many times.
static bool lora_by_waves(const LoraDev& d) { return (uint64_t)d.n_tokens * d.down * d.n <= 1u << 25; }

template <int MODE>
static void launch_down(const DownArgs& a, hipStream_t st) {
    // A tile by 16 rows where three rounds of the chip's compute units hold those, for the wait of each chunk is what counts then;
    // by 32 beyond, for half the reads of x (us of lora_add, 16 rows / 32 / 64; tokens, rank, n, outputs: f32 1691, 72, 1664, 1328
    // 27.3 / 34.5 / 40.8, 8192, 16, 4096, 2048 63 / 70 / 100, 4003, 64, 2048, 2560 59.2 / 58.2 / 64.9, 4003, 128, 2048, 512 61 / 54 /
    // 64; f16 700, 32, 1536, 2048 12.7 / 13.6 / 15.2, 4003, 64, 2048, 2560 47.6 / 43.8 / 43.3). 32 tokens a tile took 0 to 40 %
    // longer in nearly all of them, at most 2 % less.
    const uint32_t tokens = (a.l.n_tokens + 15) / 16, rows = (a.l.down + 15) / 16;
    if ((uint64_t)tokens * rows <= 3 * device_cus())
        G4_LAUNCH((k_lora_down<MODE, 1>), dim3(tokens, rows), dim3(kDownWaves * 64), 0, st, a);
    else
        G4_LAUNCH((k_lora_down<MODE, 2>), dim3(tokens, (rows + 1) / 2), dim3(kDownWaves * 64), 0, st, a);
}
template <uint32_t XT>
static void launch_down_few(const DownArgs& a, hipStream_t st) {
    const dim3 grid(a.l.n_tokens, (a.l.down + kFewRows * kFewWaves - 1) / (kFewRows * kFewWaves));
    if (a.a_type == G4_BF16) G4_LAUNCH((k_lora_down_few<XT, true>), grid, dim3(kFewWaves * 64), 0, st, a);
    else G4_LAUNCH((k_lora_down_few<XT, false>), grid, dim3(kFewWaves * 64), 0, st, a);
}

void lora_launch_down(const LoraDev& d, uint32_t lora_type, const void* x, uint32_t x_type, uint64_t x_stride,
                      const float* x_scales, hipStream_t st) {
    const DownArgs a = {d, x, x_scales, x_stride, x_type, lora_type};
    if (lora_by_waves(d)) {
        if (x_type == G4_F32) launch_down_few<G4_F32>(a, st);
        else if (x_type == G4_F16) launch_down_few<G4_F16>(a, st);
        else if (x_type == G4_BF16) launch_down_few<G4_BF16>(a, st);
        else launch_down_few<G4_E4M3>(a, st);
    } else if (x_type == G4_E4M3) {
        if (lora_type == G4_F16) launch_down<kDownE4m3F16>(a, st);
        else launch_down<kDownE4m3Bf16>(a, st);
    } else if (x_type == lora_type) {
        if (lora_type == G4_F16) launch_down<kDownF16>(a, st);
        else launch_down<kDownBf16>(a, st);
    } else if (x_type == G4_F32) {
        launch_down<kDownF32>(a, st);
    } else {
        launch_down<kDownMixed>(a, st);
    }
}

}  // namespace g4

using namespace g4;

extern "C" {

int g4_lora_workspace_size(const g4_lora* lora, uint32_t n_tokens, size_t* bytes) {
    if (!bytes) return fail(G4_EINVAL, "g4_lora_workspace_size: bytes is NULL");
    const int rc = lora_check("loraAdd", lora);
    if (rc) return rc;
    if (n_tokens > kMaxRows) return fail(G4_EINVAL, "loraAdd: %u tokens (at most 2^22)", n_tokens);
    *bytes = lora_bytes(lora, n_tokens);
    return G4_OK;
}

int g4_lora_add(const g4_lora* lora, const int32_t* adapter_ids, const void* x, const float* x_scales, const void* base,
                void* out, const g4_lora_add_params* p, void* workspace, size_t workspace_bytes, void* stream) {
    const char* what = "loraAdd";
    if (!p) return fail(G4_EINVAL, "%s: NULL params", what);
    const int rc = lora_check(what, lora);
    if (rc) return rc;
    if (p->n_tokens > kMaxRows) return fail(G4_EINVAL, "%s: %u tokens (at most 2^22)", what, p->n_tokens);
    if (p->x_type > G4_E4M3) return fail(G4_EINVAL, "%s: x_type %u", what, p->x_type);
    if (p->out_type > G4_BF16) return fail(G4_EINVAL, "%s: out_type %u (f32, f16 or bf16)", what, p->out_type);
    if (p->reserved) return fail(G4_EINVAL, "%s: reserved must be 0", what);
    if (!adapter_ids || !x || !base || !out || !workspace)
        return fail(G4_EINVAL, "%s: NULL adapter_ids, x, base, out or workspace", what);
    if (!x_scales != (p->x_type != G4_E4M3)) return fail(G4_EINVAL, "%s: x_scales go with an e4m3 x", what);
    LoraDev d = lora_dev(lora, p->n_tokens);
    const uint64_t xs = p->x_stride ? p->x_stride : d.n, bs = p->base_stride ? p->base_stride : d.rows,
                   os = p->out_stride ? p->out_stride : d.rows;
    if (xs < d.n || bs < d.rows || os < d.rows) return fail(G4_EINVAL, "%s: a stride is below its row", what);
    if (xs > (1ull << 40) || bs > (1ull << 40) || os > (1ull << 40)) return fail(G4_EINVAL, "%s: a stride is too long", what);
    if (base == out && bs != os && p->n_tokens > 1) return fail(G4_EINVAL, "%s: base may be out with one stride only", what);
    if (!aligned(x, 16) || xs * type_bytes(p->x_type) % 16) return fail(G4_EINVAL, "%s: x's rows must be 16-byte aligned", what);
    const uint32_t width = type_bytes(p->out_type);
    if (!aligned(base, width) || !aligned(out, width) || !aligned(adapter_ids, 4) || !aligned(x_scales, 4))
        return fail(G4_EINVAL, "%s: misaligned adapter_ids, x_scales, base or out", what);
    if (!aligned(workspace, 16)) return fail(G4_EINVAL, "%s: workspace must be 16-byte aligned", what);
    if (workspace_bytes < lora_bytes(lora, p->n_tokens)) return fail(G4_ENOSPC, "%s: workspace too small", what);
    if (p->n_tokens == 0) return G4_OK;
    d.ids = adapter_ids;
    d.u = static_cast<float*>(workspace);
    // The down product is done with x before out is written.
    const LoraOperands l = lora_operands(d);
    const Operand o_x = rows_operand("x", x, p->x_type, d.n, xs, p->n_tokens),
                  o_xs = {"x_scales", one_range(x_scales, 4ull * p->n_tokens)},
                  o_base = rows_operand("base", base, p->out_type, d.rows, bs, p->n_tokens),
                  o_out = rows_operand("out", out, p->out_type, d.rows, os, p->n_tokens);
    int meet = apart_check(what, l.u, {o_x, o_xs, l.a, l.b, l.scales, l.ids, o_base, o_out});
    if (!meet) meet = apart_check(what, o_out, {out == base ? Operand{} : o_base, l.b, l.scales, l.ids});
    if (meet) return meet;
    lora_launch_down(d, lora->type, x, p->x_type, xs, x_scales, as_stream(stream));
    G4_CHECK_LAUNCH("k_lora_down");
    UpArgs a = {};
    a.l = d;
    a.base = base;
    a.out = out;
    a.base_stride = bs;
    a.out_stride = os;
    a.type = p->out_type;
    auto launch = [&](auto tiles) {
        constexpr int TILES = decltype(tiles)::value, per = 16 * TILES * kUpWaves;
        const dim3 grid((p->n_tokens + 15) / 16, (d.rows + per - 1) / per), block(kUpWaves * 64);
        if (lora->type == G4_F16) G4_LAUNCH((k_lora_up<TILES, false>), grid, block, 0, as_stream(stream), a);
        else G4_LAUNCH((k_lora_up<TILES, true>), grid, block, 0, as_stream(stream), a);
    };
    // Few tokens: more waves, each waiting for less; many: a token's sums serve four tiles (us, 2560 outputs, rank 16, one
    // tile a wave / four: 64 tokens 6.8 / 10.6, 256 7.0 / 7.4, 512 9.0 / 8.7, 4096 34.5 / 28.5).
    if (p->n_tokens <= 256) launch(std::integral_constant<int, 1>{});
    else launch(std::integral_constant<int, 4>{});
    G4_CHECK_LAUNCH("k_lora_up");
    return G4_OK;
}

}  // extern "C"
