// Projections of a served batch in 8 bits (g4_linear_e4m3):
//   out[t][o] = x_scales[t] * weight_scales[o] * sum_k x[t][k] weight[o][k]
// and, in the same launch's epilogue, the requests' low-rank adapters (lora.h).
//
// The 8-bit MFMA adds the products of a group with 13 bits below the largest of them (measured over random
// rows: a sum of 128 is off by 1.4e-5 of itself, at most 2^-12.3 of the largest product). Elements widened to
// f16, which is exact, give sums in f32. Weight rows are the matrix operand's rows, tokens its columns: a lane
// ends with four consecutive outputs of one token.
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
    uint32_t out_type, wide, low;  // low: 0 no adapters, else their type
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
// Eight of them (q: 0 to 3) as f16, exactly.
__device__ __forceinline__ f16x8 widen8(const Row32& r, int q) {
    f16x8 h;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const uint32_t w = r.v[q / 2][2 * (q & 1) + i];
        const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false), hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true);
        h[4 * i] = lo[0];
        h[4 * i + 1] = lo[1];
        h[4 * i + 2] = hi[0];
        h[4 * i + 3] = hi[1];
    }
    return h;
}

// Sums of one 16-output tile: scales, adapters, the store.
__device__ __forceinline__ void finish(const Linear8Args& a, f32x4 sum, unsigned o0, unsigned t) {
    const unsigned lane = threadIdx.x & 63, g = lane >> 4, o = o0 + 4 * g;
    const bool valid = t < a.n_tokens;
    const float xs = valid ? a.x_scales[t] : 0.0f;
    f32x4 acc[1];
#pragma unroll
    for (int i = 0; i < 4; i++) acc[0][i] = sum[i] * xs * (o + i < a.rows ? a.w_scales[o + i] : 0.0f);
    if (a.low) {
        const int id = lora_id(a.l, t, valid);
        if (a.low == G4_F16) lora_up<1, false>(acc, a.l, o0, t, id);
        else lora_up<1, true>(acc, a.l, o0, t, id);
    }
    if (valid && o < a.rows) store4(a.out, a.out_type, t * a.out_stride + o, acc[0], a.wide, a.rows - o);
}

// Few tokens: 16 outputs by 16 CT tokens a workgroup, its waves take every Wth 128 of k.
template <int CT, int W>
__global__ __launch_bounds__(W * 64) void k_linear8_few(const Linear8Args a) {
    __shared__ f32x4 s_sum[W][CT][64];
    const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
    const unsigned o0 = blockIdx.y * 16, t0 = blockIdx.x * (16 * CT);
    const uint8_t* w = a.w + (uint64_t)min(o0 + col, a.rows - 1) * a.n;
    f32x4 acc[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ct++) acc[ct] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (unsigned k0 = wave * 128; k0 < a.n; k0 += W * 128) {
        const unsigned k = k0 + 32 * g;
        const Row32 wv = row32(w, k, a.n);
        f16x8 wh[4];
#pragma unroll
        for (int q = 0; q < 4; q++) wh[q] = widen8(wv, q);
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            const unsigned t = min(t0 + 16 * ct + col, a.n_tokens - 1);
            const Row32 xv = row32(a.x + t * a.x_stride, k, a.n);
#pragma unroll
            for (int q = 0; q < 4; q++) acc[ct] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wh[q], widen8(xv, q), acc[ct], 0, 0, 0);
        }
    }
#pragma unroll
    for (int ct = 0; ct < CT; ct++) s_sum[wave][ct][lane] = acc[ct];
    __syncthreads();
    for (unsigned ct = wave; ct < CT; ct += W) {
        f32x4 s = s_sum[0][ct][lane];
#pragma unroll
        for (int i = 1; i < W; i++) s += s_sum[i][ct][lane];
        finish(a, s, o0, t0 + 16 * ct + col);
    }
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
    if (p->out_type > G4_BF16) return fail(G4_EINVAL, "%s: out_type %u (f32, f16 or bf16)", what, p->out_type);
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

template <int CT, int W>
void launch_few(const Linear8Args& a, hipStream_t st) {
    G4_LAUNCH((k_linear8_few<CT, W>), dim3((a.n_tokens + 16 * CT - 1) / (16 * CT), (a.rows + 15) / 16), dim3(W * 64), 0, st, a);
}

}  // namespace

extern "C" {

int g4_linear_e4m3_workspace_size(const g4_linear_e4m3_params* p, const g4_lora* lora, size_t* bytes) {
    if (!bytes) return fail(G4_EINVAL, "g4_linear_e4m3_workspace_size: bytes is NULL");
    const int rc = linear8_check(p, lora);
    if (rc) return rc;
    *bytes = 16 + (lora ? lora_most_bytes(lora, p->n_tokens) : 0);
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
    const uint32_t width = type_bytes(p->out_type);
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
    a.out_type = p->out_type;
    a.wide = aligned(out, 4 * width) && os % 4 == 0;
    const hipStream_t st = as_stream(stream);
    if (lora) {
        a.low = lora->type;
        a.l = lora_dev(lora, p->n_tokens);
        a.l.ids = adapter_ids;
        a.l.u = static_cast<float*>(workspace);
        lora_launch_down(a.l, lora->type, x, G4_E4M3, xs, x_scales, st);
        G4_CHECK_LAUNCH("k_lora_down");
    }
    if (p->n_tokens <= 16) launch_few<1, 4>(a, st);
    else launch_few<4, 4>(a, st);
    G4_CHECK_LAUNCH("k_linear8");
    return G4_OK;
}

}  // extern "C"
