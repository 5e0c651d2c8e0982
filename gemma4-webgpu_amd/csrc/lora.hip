// Low-rank adapters of many requests beside a projection made elsewhere
// (g4_lora_add), and the down product that linear8.hip shares.
#include "lora.h"

namespace g4 {

// How x and the adapters' rows meet. 16-bit products are exact in f32, and so is an e4m3 element as f16 or bf16; other
// pairs are widened to f32.
enum { kDownF16, kDownBf16, kDownE4m3F16, kDownE4m3Bf16, kDownF32 };

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
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[w], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[w], true);
        if constexpr (BF) {
            r[2 * w] = (uint32_t)f2bf(lo[0]) | (uint32_t)f2bf(lo[1]) << 16;
            r[2 * w + 1] = (uint32_t)f2bf(hi[0]) | (uint32_t)f2bf(hi[1]) << 16;
        } else {
            r[2 * w] = (uint32_t)f2h(lo[0]) | (uint32_t)f2h(lo[1]) << 16;
            r[2 * w + 1] = (uint32_t)f2h(hi[0]) | (uint32_t)f2h(hi[1]) << 16;
        }
    }
    return r;
}

constexpr int kDownWaves = 4;

// 16 CT tokens by groups of RT 16-row tiles of the adapters' down rows; blockIdx: (token tile, piece of k, which of the
// tile's adapters). The four waves take every fourth 64-element chunk of the piece.
template <int MODE, int CT, int RT>
__global__ __launch_bounds__(kDownWaves * 64) void k_lora_down(const DownArgs a) {
    __shared__ f32x4 s_sum[kDownWaves][RT * CT][64];
    __shared__ int s_id[64];
    const LoraDev& l = a.l;
    const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
    const unsigned t0 = blockIdx.x * (16 * CT);
    // Lane: token of the tile. One wave's reading for all, so that they agree whatever happens to the array meanwhile.
    if (wave == 0) s_id[lane] = lora_id(l, t0 + lane, lane < 16 * CT && t0 + lane < l.n_tokens);
    __syncthreads();
    const int id = s_id[lane];
    uint64_t left = __ballot(id >= 0);
    const unsigned chunks = (l.n + 63) / 64;
    unsigned nth = 0;
    while (left) {  // uniform over the workgroup
        const int ad = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
        const uint64_t with = __ballot(id == ad);
        left &= ~with;
        if (nth++ % gridDim.z != blockIdx.z) continue;
        for (unsigned r0 = 0; r0 < l.down; r0 += 16 * RT) {
            f32x4 acc[RT][CT];
#pragma unroll
            for (int rt = 0; rt < RT; rt++)
#pragma unroll
                for (int ct = 0; ct < CT; ct++) acc[rt][ct] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            for (unsigned c = blockIdx.y * kDownWaves + wave; c < chunks; c += gridDim.y * kDownWaves) {
                const unsigned k = c * 64 + g * 16;  // the lane's 16 elements
                const bool in = k < l.n;
                if constexpr (MODE == kDownF32) {
                    f32x4 w[RT][4];
#pragma unroll
                    for (int rt = 0; rt < RT; rt++) {
                        const unsigned row = min(r0 + 16 * rt + col, l.down - 1);
                        const uint64_t at = ((uint64_t)ad * l.down + row) * l.n + k;
#pragma unroll
                        for (int q = 0; q < 4; q++) w[rt][q] = in ? load4(l.a, a.a_type, at + 4 * q, true, 4) : f32x4{0, 0, 0, 0};
                    }
#pragma unroll
                    for (int ct = 0; ct < CT; ct++) {
                        if (!((with >> (16 * ct)) & 0xFFFF)) continue;
                        const unsigned t = min(t0 + 16 * ct + col, l.n_tokens - 1);
                        f32x4 x[4];
#pragma unroll
                        for (int q = 0; q < 4; q++)
                            x[q] = in ? load4(a.x, a.x_type, t * a.x_stride + k + 4 * q, true, 4) : f32x4{0, 0, 0, 0};
#pragma unroll
                        for (int rt = 0; rt < RT; rt++)
#pragma unroll
                            for (int e = 0; e < 16; e++)
                                acc[rt][ct] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[rt][e / 4][e % 4], x[e / 4][e % 4], acc[rt][ct], 0, 0, 0);
                    }
                } else {
                    constexpr bool BF = MODE == kDownBf16 || MODE == kDownE4m3Bf16;
                    u32x4 w[RT][2];
#pragma unroll
                    for (int rt = 0; rt < RT; rt++) {
                        const unsigned row = min(r0 + 16 * rt + col, l.down - 1);
                        const uint16_t* p = static_cast<const uint16_t*>(l.a) + ((uint64_t)ad * l.down + row) * l.n + k;
                        w[rt][0] = in ? ldg<u32x4>(p) : u32x4{0, 0, 0, 0};
                        w[rt][1] = in ? ldg<u32x4>(p + 8) : u32x4{0, 0, 0, 0};
                    }
#pragma unroll
                    for (int ct = 0; ct < CT; ct++) {
                        if (!((with >> (16 * ct)) & 0xFFFF)) continue;
                        const unsigned t = min(t0 + 16 * ct + col, l.n_tokens - 1);
                        u32x4 x[2];
                        if constexpr (MODE == kDownE4m3F16 || MODE == kDownE4m3Bf16) {
                            const u32x4 q = in ? ldg<u32x4>(static_cast<const uint8_t*>(a.x) + t * a.x_stride + k) : u32x4{0, 0, 0, 0};
                            x[0] = e4m3_wide<BF>(u32x2{q[0], q[1]});
                            x[1] = e4m3_wide<BF>(u32x2{q[2], q[3]});
                        } else {
                            const uint16_t* p = static_cast<const uint16_t*>(a.x) + t * a.x_stride + k;
                            x[0] = in ? ldg<u32x4>(p) : u32x4{0, 0, 0, 0};
                            x[1] = in ? ldg<u32x4>(p + 8) : u32x4{0, 0, 0, 0};
                        }
#pragma unroll
                        for (int rt = 0; rt < RT; rt++)
#pragma unroll
                            for (int h = 0; h < 2; h++) {
                                if constexpr (BF)
                                    acc[rt][ct] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                        __builtin_bit_cast(bf16x8, w[rt][h]), __builtin_bit_cast(bf16x8, x[h]), acc[rt][ct], 0, 0, 0);
                                else
                                    acc[rt][ct] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                        __builtin_bit_cast(f16x8, w[rt][h]), __builtin_bit_cast(f16x8, x[h]), acc[rt][ct], 0, 0, 0);
                            }
                    }
                }
            }
#pragma unroll
            for (int rt = 0; rt < RT; rt++)
#pragma unroll
                for (int ct = 0; ct < CT; ct++) s_sum[wave][rt * CT + ct][lane] = acc[rt][ct];
            __syncthreads();
            for (unsigned i = wave; i < RT * CT; i += kDownWaves) {
                const unsigned rt = i / CT, ct = i % CT, t = t0 + 16 * ct + col, row = r0 + 16 * rt + 4 * g;
                f32x4 s = s_sum[0][i][lane];
#pragma unroll
                for (int w = 1; w < kDownWaves; w++) s += s_sum[w][i][lane];
                if (((with >> (16 * ct + col)) & 1) && row < l.down) {  // down and row: multiples of 4
                    if (a.x_scales) s *= a.x_scales[t];
                    stg<f32x4>(l.u + ((uint64_t)blockIdx.y * l.n_tokens + t) * l.down + row, s);
                }
            }
            __syncthreads();
        }
    }
}

// out = base + the adapters' part. A wave: 16 tokens by 64 outputs.
constexpr int kUpTiles = 4, kUpWaves = 4;
struct UpArgs {
    LoraDev l;
    const void* base;  // may be out
    void* out;
    uint64_t base_stride, out_stride;
    uint32_t type, wide;
};
template <bool BF>
__global__ __launch_bounds__(kUpWaves * 64) void k_lora_up(const UpArgs a) {
    const LoraDev& l = a.l;
    const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
    const unsigned t = blockIdx.x * 16 + (lane & 15), o0 = (blockIdx.y * kUpWaves + wave) * (16 * kUpTiles);
    if (o0 >= l.rows) return;
    const bool valid = t < l.n_tokens;
    const int id = lora_id(l, t, valid);
    f32x4 acc[kUpTiles];
#pragma unroll
    for (int rt = 0; rt < kUpTiles; rt++) {
        const unsigned o = o0 + 16 * rt + 4 * g;
        acc[rt] = valid && o < l.rows ? load4(a.base, a.type, t * a.base_stride + o, a.wide, l.rows - o) : f32x4{0, 0, 0, 0};
    }
    lora_up<16, kUpTiles, BF>(l, o0, t, id, [&](int rt, int i, float v) __attribute__((always_inline)) { acc[rt][i] += v; });
#pragma unroll
    for (int rt = 0; rt < kUpTiles; rt++) {
        const unsigned o = o0 + 16 * rt + 4 * g;
        if (valid && o < l.rows) store4(a.out, a.type, t * a.out_stride + o, acc[rt], a.wide, l.rows - o);
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
    d.splits = lora_splits(l, n_tokens);
    return d;
}

uint32_t lora_splits(const g4_lora* l, uint32_t n_tokens) {
    if (n_tokens == 0) return 1;
    const uint32_t per = n_tokens > 256 ? 64 : 16, tiles = (n_tokens + per - 1) / per, chunks = (l->n + 63) / 64;
    uint32_t splits = (chunks + kDownWaves - 1) / kDownWaves;  // a chunk a wave at least
    const uint32_t fill = (device_cus() + tiles - 1) / tiles;
    if (splits > fill) splits = fill;
    if (splits > 8) splits = 8;
    return splits;
}
size_t lora_bytes(const g4_lora* l, uint32_t n_tokens) {
    return ((size_t)lora_splits(l, n_tokens) * n_tokens * l->n_segs * l->rank * 4 + 15) & ~(size_t)15;
}
// splits * n <= 64 (CUs + tiles - 1) for every n up to n_tokens, and splits <= 8.
size_t lora_most_bytes(const g4_lora* l, uint32_t n_tokens) {
    const uint64_t few = 8ull * n_tokens, many = 64ull * device_cus() + n_tokens + 64;
    return (size_t)(few < many ? few : many) * l->n_segs * l->rank * 4 + 16;
}

template <int MODE>
static void launch_down(const DownArgs& a, hipStream_t st) {
    const uint32_t T = a.l.n_tokens;
    if (T > 256) {
        G4_LAUNCH((k_lora_down<MODE, 4, 2>), dim3((T + 63) / 64, a.l.splits, 1), dim3(kDownWaves * 64), 0, st, a);
    } else {
        G4_LAUNCH((k_lora_down<MODE, 1, 4>), dim3((T + 15) / 16, a.l.splits, T < 16 ? T : 16), dim3(kDownWaves * 64), 0, st, a);
    }
}

void lora_launch_down(const LoraDev& d, uint32_t lora_type, const void* x, uint32_t x_type, uint64_t x_stride,
                      const float* x_scales, hipStream_t st) {
    DownArgs a = {d, x, x_scales, x_stride, x_type, lora_type};
    if (x_type == G4_E4M3) {
        if (lora_type == G4_F16) launch_down<kDownE4m3F16>(a, st);
        else launch_down<kDownE4m3Bf16>(a, st);
    } else if (x_type == lora_type) {
        if (lora_type == G4_F16) launch_down<kDownF16>(a, st);
        else launch_down<kDownBf16>(a, st);
    } else {
        launch_down<kDownF32>(a, st);
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
    *bytes = lora_most_bytes(lora, n_tokens);
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
    if (!aligned(x, 16) || xs * type_bytes(p->x_type) % 16) return fail(G4_EINVAL, "%s: x's rows must be 16-byte aligned", what);
    const uint32_t width = type_bytes(p->out_type);
    if (!aligned(base, width) || !aligned(out, width) || !aligned(adapter_ids, 4) || !aligned(x_scales, 4))
        return fail(G4_EINVAL, "%s: misaligned adapter_ids, x_scales, base or out", what);
    if (!aligned(workspace, 16)) return fail(G4_EINVAL, "%s: workspace must be 16-byte aligned", what);
    if (workspace_bytes < lora_bytes(lora, p->n_tokens)) return fail(G4_ENOSPC, "%s: workspace too small", what);
    if (p->n_tokens == 0) return G4_OK;
    d.ids = adapter_ids;
    d.u = static_cast<float*>(workspace);
    lora_launch_down(d, lora->type, x, p->x_type, xs, x_scales, as_stream(stream));
    G4_CHECK_LAUNCH("k_lora_down");
    UpArgs a = {};
    a.l = d;
    a.base = base;
    a.out = out;
    a.base_stride = bs;
    a.out_stride = os;
    a.type = p->out_type;
    a.wide = aligned(base, 4 * width) && aligned(out, 4 * width) && bs % 4 == 0 && os % 4 == 0;
    const dim3 grid((p->n_tokens + 15) / 16, (d.rows + 16 * kUpTiles * kUpWaves - 1) / (16 * kUpTiles * kUpWaves));
    if (lora->type == G4_F16) G4_LAUNCH((k_lora_up<false>), grid, dim3(kUpWaves * 64), 0, as_stream(stream), a);
    else G4_LAUNCH((k_lora_up<true>), grid, dim3(kUpWaves * 64), 0, as_stream(stream), a);
    G4_CHECK_LAUNCH("k_lora_up");
    return G4_OK;
}

}  // extern "C"
