// A batch's rows between two blocks (g4_add_rms_norm, g4_quantize_rows): the
// branch's own norm, the residual's addition, the next block's norm, and the
// rows in 8 bits for the projections (linear8.hip), in one pass.
//
// b = x * w1 / sqrt(mean x^2 + eps) (or x);  r = residual + b, rounded to the residual's type;
// y = r * w2 / sqrt(mean r^2 + eps);  s = max|y| / 448, codes e4m3(y / s).
//
// Bound by the bytes: a row is loaded once into registers, and every sum works on
// those. The largest |y| is the largest |r w2| times one factor, so the second
// norm and the scale share one reduction, and a row of one wave has no barrier
// at all. Everything a row needs is requested before its first sum; the operands'
// widths are compiled in, so that 16-bit ones take half the registers and more rows
// are under way (types told apart at run time, as with f32 weights: 68 us below).
//
// Measured (a copy reaches 5.0 TB/s here): 8191 rows of 5376, 16 bits in, sum out, e4m3 out, 61 us, 5.1 TB/s;
// 4096 rows of 1536, f32 in, both norms, 15.2 us; 4000 attention outputs of 2048 in 8 bits 8.2 us; one row
// 2.9 us, the launch and two chains of loads and sums. Rows that are not aligned to 16 bytes, or whose n is no multiple of
// 8, go an element a load and store: 8191 rows of 5375, 16 bits, 202 us (5376: 61 to 69), 4096 of 1535, f32, 27.5 (20 with other
// rows each time), quantized rows of 2047 11.4 (8.6). Rows above 16384 elements do too: 2048 of 32768, f32, 247 (173 of bytes).
#include <type_traits>

#include "decode_core.h"
#include "launch_rules.h"
#include "rows.h"

namespace g4 {

struct NormRowsArgs {
    const void* x;            // may be out
    const void* residual;     // may be residual_out
    const void* __restrict__ post;
    const void* __restrict__ weight;
    void* residual_out;
    void* out;
    float* __restrict__ scales;
    uint64_t x_stride, residual_stride, residual_out_stride, out_stride;
    uint32_t rows, n;
    uint32_t x_type, residual_type, weight_type, out_type;
    float eps, inv_n;
    uint32_t norm;            // 0: y = r
};

template <int CTRL>
__device__ __forceinline__ uint32_t nr_dpp(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, CTRL, 0xf, 0xf, false);
}
__device__ __forceinline__ float nr_wave_sum(float x) {  // in every lane: 16-lane rotations, then rows and halves swapped
    x += __uint_as_float(nr_dpp<0x128>(__float_as_uint(x)));
    x += __uint_as_float(nr_dpp<0x124>(__float_as_uint(x)));
    x += __uint_as_float(nr_dpp<0x122>(__float_as_uint(x)));
    x += __uint_as_float(nr_dpp<0x121>(__float_as_uint(x)));
    return add_xor32(add_xor16(x));
}
// The largest magnitude, as its bits: a NaN's are above every number's.
__device__ __forceinline__ uint32_t nr_wave_top(uint32_t x) {
    x = max(x, nr_dpp<0x128>(x));
    x = max(x, nr_dpp<0x124>(x));
    x = max(x, nr_dpp<0x122>(x));
    x = max(x, nr_dpp<0x121>(x));
    auto sw = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max(sw[0], sw[1]);
    sw = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return max(sw[0], sw[1]);
}

// Sum and largest magnitude over the W waves of a row.
template <int W>
__device__ __forceinline__ void nr_reduce(float& sum, uint32_t& top, float (&s_sum)[W], uint32_t (&s_top)[W]) {
    sum = nr_wave_sum(sum);
    top = nr_wave_top(top);
    if constexpr (W > 1) {
        const unsigned wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) {
            s_sum[wave] = sum;
            s_top[wave] = top;
        }
        __syncthreads();
        sum = 0.0f;
        top = 0;
#pragma unroll
        for (int i = 0; i < W; i++) {
            sum += s_sum[i];
            top = max(top, s_top[i]);
        }
    }
}

// NV * 8 elements of a row as they lie: 16-bit ones fill the first half of each eight. Elements past n are 0. Element i of a
// thread is (i / 8 * TPR + t) * 8 + i % 8 of the row with VEC, else i * TPR + t. WIDTH: the bytes of an element, 0 known
// only at run time (with the registers of four).
template <int NV, int WIDTH>
struct RawRow {
    u32x4 a[NV], b[WIDTH == 2 ? 1 : NV];
};
template <int TPR, int NV, bool VEC, int WIDTH>
__device__ __forceinline__ RawRow<NV, WIDTH> nr_load(const void* p, uint32_t type, unsigned t, unsigned n) {
    RawRow<NV, WIDTH> r;
    const char* base = static_cast<const char*>(p);
    const bool full = WIDTH == 0 ? type == G4_F32 : WIDTH == 4;
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const unsigned at = (i * TPR + t) * 8;
            u32x4 a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
            if (at < n) a = ldg<u32x4>(base + (full ? 4 * at : 2 * at));
            if (at < n && full) b = ldg<u32x4>(base + 4 * at + 16);
            r.a[i] = a;
            if constexpr (WIDTH != 2) r.b[i] = b;
        }
    } else {
        static_assert(WIDTH == 0, "one element a load: any type");
        uint32_t e[NV * 8];
#pragma unroll
        for (int i = 0; i < NV * 8; i++) {
            const unsigned at = i * TPR + t;
            uint32_t v = 0;
            if (at < n && full) v = ldg<uint32_t>(base + 4 * at);
            if (at < n && !full) v = ldg<uint16_t>(base + 2 * at);
            e[i] = v;
        }
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const uint32_t* q = e + 8 * i;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                r.a[i][j] = full ? q[j] : q[2 * j] | q[2 * j + 1] << 16;
                r.b[i][j] = q[4 + j];
            }
        }
    }
    return r;
}
// f(i, element i).
template <int NV, int WIDTH, typename F>
__device__ __forceinline__ void nr_each(const RawRow<NV, WIDTH>& r, uint32_t type, F&& f) {
#pragma unroll
    for (int i = 0; i < NV * 8; i++) {
        const uint32_t pair = r.a[i / 8][i % 8 / 2], word = WIDTH == 2 ? 0 : i % 8 < 4 ? r.a[i / 8][i % 4] : r.b[WIDTH == 2 ? 0 : i / 8][i % 4];
        const float h = h2f((uint16_t)(pair >> (16 * (i & 1)))), b = __uint_as_float((i & 1) ? pair & 0xFFFF0000u : pair << 16);
        const float half = type == G4_F16 ? h : b;
        f(i, WIDTH == 4 ? __uint_as_float(word) : WIDTH == 2 ? half : type == G4_F32 ? __uint_as_float(word) : half);
    }
}
template <int E>
__device__ __forceinline__ void nr_round(float (&v)[E], uint32_t type) {
    if (type == G4_F16) {
#pragma unroll
        for (int i = 0; i < E; i++) v[i] = h2f(f2h(v[i]));
    } else if (type == G4_BF16) {
#pragma unroll
        for (int i = 0; i < E; i++) v[i] = bf2f(f2bf(v[i]));
    }
}
template <int TPR, int NV, bool VEC>
__device__ __forceinline__ void nr_store(const float (&v)[NV * 8], void* p, uint32_t type, unsigned t, unsigned n) {
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const unsigned at = (i * TPR + t) * 8;
            if (at >= n) continue;
            if (type == G4_F32) {
                stg<f32x4>(static_cast<float*>(p) + at, f32x4{v[8 * i], v[8 * i + 1], v[8 * i + 2], v[8 * i + 3]});
                stg<f32x4>(static_cast<float*>(p) + at + 4, f32x4{v[8 * i + 4], v[8 * i + 5], v[8 * i + 6], v[8 * i + 7]});
            } else if (type == G4_E4M3) {
                u32x2 q;
#pragma unroll
                for (int e = 0; e < 2; e++)
                    q[e] = e4m3_pair(v[8 * i + 4 * e], v[8 * i + 4 * e + 1]) |
                           e4m3_pair(v[8 * i + 4 * e + 2], v[8 * i + 4 * e + 3]) << 16;
                stg<u32x2>(static_cast<uint8_t*>(p) + at, q);
            } else {
                u32x4 q;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float a = v[8 * i + 2 * e], b = v[8 * i + 2 * e + 1];
                    q[e] = type == G4_F16 ? (uint32_t)f2h(a) | (uint32_t)f2h(b) << 16 : (uint32_t)f2bf(a) | (uint32_t)f2bf(b) << 16;
                }
                stg<u32x4>(static_cast<uint16_t*>(p) + at, q);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV * 8; i++) {
            const unsigned at = i * TPR + t;
            if (at >= n) continue;
            if (type == G4_F32) stg<float>(static_cast<float*>(p) + at, v[i]);
            else if (type == G4_E4M3) stg<uint8_t>(static_cast<uint8_t*>(p) + at, (uint8_t)e4m3_pair(v[i], 0.0f));
            else stg<uint16_t>(static_cast<uint16_t*>(p) + at, type == G4_F16 ? f2h(v[i]) : f2bf(v[i]));
        }
    }
}

__device__ __forceinline__ const void* nr_row(const void* p, uint32_t type, uint64_t at) {
    return static_cast<const char*>(p) + at * (type == G4_F32 ? 4 : type == G4_E4M3 ? 1 : 2);
}

// TPR threads a row, NV * 8 elements a thread. VEC: 8 elements a load (16 or 32 bytes; rows aligned, n a multiple of 8).
// XW, RW, WW: the widths of x, the residual and the weights.
template <int TPR, int NV, bool VEC, int XW, int RW, int WW>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void k_norm_rows(const NormRowsArgs a) {
    constexpr int E = NV * 8, W = TPR / 64;
    constexpr bool LATE = TPR == 1024;  // 128 registers a wave: each operand only when the one before is done with
    __shared__ float s_sum[2][W];
    __shared__ uint32_t s_top[2][W];
    const unsigned group = TPR == 1024 ? blockIdx.y * gridDim.x + blockIdx.x : blockIdx.x;
    const unsigned row = TPR < 256 ? group * (256 / TPR) + threadIdx.x / TPR : group;
    const unsigned t = TPR < 256 ? threadIdx.x % TPR : threadIdx.x;
    if (row >= a.rows) return;  // whole waves, of a kernel without barriers
    const unsigned n = a.n;
    auto load_residual = [&]() __attribute__((always_inline)) {
        return nr_load<TPR, NV, VEC, RW>(nr_row(a.residual, a.residual_type, row * a.residual_stride), a.residual_type, t, n);
    };
    const auto x = nr_load<TPR, NV, VEC, XW>(nr_row(a.x, a.x_type, row * a.x_stride), a.x_type, t, n);
    RawRow<NV, RW> res = {};
    if (!LATE && a.residual) res = load_residual();
    // The next norm's weights are requested early too: behind the sums they would be waited for.
    RawRow<NV, WW> w2 = {};
    if (!LATE && a.weight) w2 = nr_load<TPR, NV, VEC, WW>(a.weight, a.weight_type, t, n);
    float v[E];
    nr_each(x, a.x_type, [&](int i, float e) __attribute__((always_inline)) { v[i] = e; });
    if (a.post) {
        float sum = 0.0f;
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < E; i++) sum = __builtin_fmaf(v[i], v[i], sum);
        const auto w = nr_load<TPR, NV, VEC, WW>(a.post, a.weight_type, t, n);
        nr_reduce<W>(sum, top, s_sum[0], s_top[0]);
        const float inv = 1.0f / sqrtf(sum * a.inv_n + a.eps);
        nr_each(w, a.weight_type, [&](int i, float e) __attribute__((always_inline)) { v[i] *= e * inv; });
    }
    auto add = [&](int i, float e) __attribute__((always_inline)) { v[i] += e; };
    if constexpr (LATE) {
        if (a.residual) nr_each(load_residual(), a.residual_type, add);
    } else {
        if (a.residual) nr_each(res, a.residual_type, add);
    }
    if (a.residual || a.residual_out) nr_round<E>(v, a.residual_type);
    if (a.residual_out)
        nr_store<TPR, NV, VEC>(v, const_cast<void*>(nr_row(a.residual_out, a.residual_type, row * a.residual_out_stride)),
                               a.residual_type, t, n);
    if (!a.out) return;
    float sum = 0.0f, inv = 1.0f;
    uint32_t top = 0;
    if (a.norm) {
#pragma unroll
        for (int i = 0; i < E; i++) sum = __builtin_fmaf(v[i], v[i], sum);
    }
    if (a.weight) {
        auto times = [&](int i, float e) __attribute__((always_inline)) { v[i] *= e; };
        if constexpr (LATE) nr_each(nr_load<TPR, NV, VEC, WW>(a.weight, a.weight_type, t, n), a.weight_type, times);
        else nr_each(w2, a.weight_type, times);
    }
    if (a.out_type == G4_E4M3) {
#pragma unroll
        for (int i = 0; i < E; i++) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    }
    nr_reduce<W>(sum, top, s_sum[1], s_top[1]);
    if (a.norm) inv = 1.0f / sqrtf(sum * a.inv_n + a.eps);
    if (a.out_type == G4_E4M3) {
        // Rows below 2^-100 are scaled as rows of that size: 448 / top stays finite.
        const float most = fmaxf(__uint_as_float(top) * inv, 0x1p-100f);
        const bool fine = __uint_as_float(top) * inv < INFINITY;  // and no NaN
        if (t == 0) a.scales[row] = fine ? most / 448.0f : __uint_as_float(0x7FC00000u);
        const float to = 448.0f / most;
        if (!fine) {  // every code NaN
            uint8_t* o = static_cast<uint8_t*>(a.out) + row * a.out_stride;
            for (unsigned i = t; i < n; i += TPR) stg<uint8_t>(o + i, (uint8_t)0x7F);
            return;
        }
        // Both factors as one, but where their product passes f32: rows whose eps is below 3e-12, of values that small.
        if (!(inv * to < INFINITY)) {
#pragma unroll
            for (int i = 0; i < E; i++) v[i] *= inv;
            inv = 1.0f;
        }
        inv = inv * to;
    }
#pragma unroll
    for (int i = 0; i < E; i++) v[i] *= inv;
    nr_store<TPR, NV, VEC>(v, const_cast<void*>(nr_row(a.out, a.out_type, row * a.out_stride)), a.out_type, t, n);
}

constexpr uint32_t kNormMaxN = 32768;

// Eight elements a load would not fit the registers.
void launch_longest(const NormRowsArgs& a, hipStream_t st) {
    const uint32_t columns = long_row_columns(a.rows);
    G4_LAUNCH((k_norm_rows<1024, 4, false, 0, 0, 0>), dim3(columns, (a.rows + columns - 1) / columns), dim3(1024), 0, st, a);
}
template <bool VEC, int XW, int RW, int WW>
void launch_norm_rows(const NormRowsArgs& a, hipStream_t st) {
    auto launch = [&](auto tpr, auto nv) {
        constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value;
        constexpr uint32_t PER = TPR < 256 ? 256 / TPR : 1;
        const dim3 grid((a.rows + PER - 1) / PER), block(TPR * PER);
        G4_LAUNCH((k_norm_rows<TPR, NV, VEC, XW, RW, WW>), grid, block, 0, st, a);
    };
#define G4_NORM(TPR, NV) launch(std::integral_constant<int, TPR>{}, std::integral_constant<int, NV>{})
    // A wave a row where rows are short and many, else four waves a row (us, f32 with both norms into e4m3, a wave / four: rows
    // of 512: 512 of them 3.6 / 3.8, 1024 4.3 / 5.3, 16384 22.6 / 37.1; 2048 of 1024 9.1 / 10.0; of 1536: 64 4.3 / 3.5, 2048 11.4 /
    // 10.9, 16384 59.8 / 58.9).
    const bool many = a.rows >= 2 * device_cus();
    if (many && a.n <= 512) G4_NORM(64, 1);
    else if (many && a.n <= 1024) G4_NORM(64, 2);
    else if (a.n <= 2048) G4_NORM(256, 1);
    else if (a.n <= 4096) G4_NORM(256, 2);
    else if (a.n <= 6144) G4_NORM(256, 3);
    else if (a.n <= 8192) G4_NORM(256, 4);
    else if (a.n <= 16384) G4_NORM(512, 4);
    else launch_longest(a, st);
#undef G4_NORM
}
void launch_norm_rows(const NormRowsArgs& a, bool vec, hipStream_t st) {
    if (!vec) return launch_norm_rows<false, 0, 0, 0>(a, st);
    // f32 weights share one form for all types (us, weights of 16 bits / f32: 8191 rows of 5376, 16 bits, 63.4 / 68.0, with both
    // norms 70.3 / 78.7; 4096 of 1536, f32, 18.7 / 19.5, both norms 20.0 / 21.5; one row 3.3 / 3.6).
    const bool w4 = (a.post || a.weight) && a.weight_type == G4_F32, r4 = a.residual && a.residual_type == G4_F32;
    if (w4) return launch_norm_rows<true, 0, 0, 0>(a, st);
    if (a.x_type == G4_F32) return r4 ? launch_norm_rows<true, 4, 4, 2>(a, st) : launch_norm_rows<true, 4, 2, 2>(a, st);
    return r4 ? launch_norm_rows<true, 2, 4, 2>(a, st) : launch_norm_rows<true, 2, 2, 2>(a, st);
}

}  // namespace g4

using namespace g4;

namespace {

int rows_check(const char* what, uint32_t rows, uint32_t n) {
    if (rows > kMaxRows) return fail(G4_EINVAL, "%s: %u rows (at most 2^22)", what, rows);
    if (n == 0 || n > kNormMaxN) return fail(G4_EINVAL, "%s: n %u (1 to %u)", what, n, kNormMaxN);
    return G4_OK;
}
// 0 stands for rows one after the other; a row's elements are contiguous.
int stride_check(const char* what, const char* name, uint64_t& stride, uint32_t n) {
    if (stride == 0) stride = n;
    if (stride < n) return fail(G4_EINVAL, "%s: %s_stride below n %u", what, name, n);
    if (stride > (1ull << 40)) return fail(G4_EINVAL, "%s: %s_stride too long", what, name);
    return G4_OK;
}
int pointer_check(const char* what, const char* name, const void* p, uint32_t type) {
    if (!aligned(p, type_bytes(type))) return fail(G4_EINVAL, "%s: misaligned %s", what, name);
    return G4_OK;
}
// A row is stored when another may not have been read: what shares memory has to share its rows (other overlaps: apart_check).
int shared_check(const char* what, const char* names, const void* p, uint32_t p_type, uint64_t p_stride, const void* q,
                 uint32_t q_type, uint64_t q_stride, uint32_t rows) {
    if (p && p == q && (p_type != q_type || (rows > 1 && p_stride != q_stride)))
        return fail(G4_EINVAL, "%s: %s may share memory with one type and stride only", what, names);
    return G4_OK;
}
// Whether rows can be read eight elements at a time.
bool wide_rows(const void* p, uint32_t type, uint64_t stride) {
    const uint64_t to = type == G4_E4M3 ? 8 : 16;
    return !p || (aligned(p, to) && stride * type_bytes(type) % to == 0);
}

}  // namespace

extern "C" {

int g4_add_rms_norm(const void* x, const void* residual, const void* post_weight, const void* weight, void* residual_out,
                    void* out, float* scales, const g4_add_rms_norm_params* p, void* stream) {
    const char* what = "addRmsNorm";
    if (!p) return fail(G4_EINVAL, "%s: NULL params", what);
    int rc = rows_check(what, p->rows, p->n);
    if (rc) return rc;
    if (p->x_type > G4_BF16) return fail(G4_EINVAL, "%s: x_type %u (f32, f16 or bf16)", what, p->x_type);
    if (p->residual_type > G4_BF16) return fail(G4_EINVAL, "%s: residual_type %u (f32, f16 or bf16)", what, p->residual_type);
    if (p->weight_type > G4_BF16) return fail(G4_EINVAL, "%s: weight_type %u (f32, f16 or bf16)", what, p->weight_type);
    if (p->out_type > G4_E4M3) return fail(G4_EINVAL, "%s: out_type %u", what, p->out_type);
    if (p->reserved) return fail(G4_EINVAL, "%s: reserved must be 0", what);
    if (!(p->eps >= 0.0f) || p->eps > 1.0f) return fail(G4_EINVAL, "%s: eps %g (0 to 1)", what, (double)p->eps);
    if (!x) return fail(G4_EINVAL, "%s: NULL x", what);
    if (!out && !residual_out) return fail(G4_EINVAL, "%s: neither out nor residual_out", what);
    if (!out && weight) return fail(G4_EINVAL, "%s: weight without out", what);
    if (!scales != !(out && p->out_type == G4_E4M3)) return fail(G4_EINVAL, "%s: scales go with an e4m3 out", what);
    NormRowsArgs a = {};
    a.x_stride = p->x_stride;
    a.residual_stride = p->residual_stride;
    a.residual_out_stride = p->residual_out_stride;
    a.out_stride = p->out_stride;
    if ((rc = stride_check(what, "x", a.x_stride, p->n)) || (rc = stride_check(what, "residual", a.residual_stride, p->n)) ||
        (rc = stride_check(what, "residual_out", a.residual_out_stride, p->n)) ||
        (rc = stride_check(what, "out", a.out_stride, p->n)))
        return rc;
    if ((rc = pointer_check(what, "x", x, p->x_type)) || (rc = pointer_check(what, "residual", residual, p->residual_type)) ||
        (rc = pointer_check(what, "residual_out", residual_out, p->residual_type)) ||
        (rc = pointer_check(what, "post_weight", post_weight, p->weight_type)) ||
        (rc = pointer_check(what, "weight", weight, p->weight_type)) || (rc = pointer_check(what, "out", out, p->out_type)) ||
        (rc = pointer_check(what, "scales", scales, G4_F32)))
        return rc;
    if (out && out == residual_out) return fail(G4_EINVAL, "%s: out is residual_out", what);
    const uint64_t xs = a.x_stride, rs = a.residual_stride, ts = a.residual_out_stride, os = a.out_stride;
    if ((rc = shared_check(what, "out and x", out, p->out_type, os, x, p->x_type, xs, p->rows)) ||
        (rc = shared_check(what, "out and residual", out, p->out_type, os, residual, p->residual_type, rs, p->rows)) ||
        (rc = shared_check(what, "residual_out and x", residual_out, p->residual_type, ts, x, p->x_type, xs, p->rows)) ||
        (rc = shared_check(what, "residual_out and residual", residual_out, p->residual_type, ts, residual, p->residual_type, rs, p->rows)))
        return rc;
    if (p->rows == 0) return G4_OK;
    const uint64_t n = p->n, rows = p->rows;
    const Operand o_out = rows_operand("out", out, p->out_type, n, os, rows),
                  o_sum = rows_operand("residual_out", residual_out, p->residual_type, n, ts, rows),
                  o_scales = {"scales", one_range(scales, 4 * rows)};
    const Operand o_x = rows_operand("x", x, p->x_type, n, xs, rows),
                  o_res = rows_operand("residual", residual, p->residual_type, n, rs, rows),
                  o_post = rows_operand("post_weight", post_weight, p->weight_type, n, n, 1),
                  o_weight = rows_operand("weight", weight, p->weight_type, n, n, 1);
    const Operand none = {};
    if ((rc = apart_check(what, o_out, {out == x ? none : o_x, out == residual ? none : o_res, o_post, o_weight, o_sum, o_scales})) ||
        (rc = apart_check(what, o_sum, {residual_out == x ? none : o_x, residual_out == residual ? none : o_res, o_post, o_weight, o_scales})) ||
        (rc = apart_check(what, o_scales, {o_x, o_res, o_post, o_weight})))
        return rc;
    a.x = x;
    a.residual = residual;
    a.post = post_weight;
    a.weight = weight;
    a.residual_out = residual_out;
    a.out = out;
    a.scales = scales;
    a.rows = p->rows;
    a.n = p->n;
    a.x_type = p->x_type;
    a.residual_type = p->residual_type;
    a.weight_type = p->weight_type;
    a.out_type = p->out_type;
    a.eps = p->eps;
    a.inv_n = 1.0f / (float)p->n;
    a.norm = 1;
    const bool wide = p->n % 8 == 0 && wide_rows(x, a.x_type, a.x_stride) && wide_rows(residual, a.residual_type, a.residual_stride) &&
                      wide_rows(residual_out, a.residual_type, a.residual_out_stride) && wide_rows(post_weight, a.weight_type, 0) &&
                      wide_rows(weight, a.weight_type, 0) && wide_rows(out, a.out_type, a.out_stride);
    launch_norm_rows(a, wide, as_stream(stream));
    G4_CHECK_LAUNCH("k_norm_rows");
    return G4_OK;
}

int g4_quantize_rows(const void* x, uint8_t* out, float* scales, const g4_quantize_rows_params* p, void* stream) {
    const char* what = "quantizeRows";
    if (!p) return fail(G4_EINVAL, "%s: NULL params", what);
    int rc = rows_check(what, p->rows, p->n);
    if (rc) return rc;
    if (p->x_type > G4_BF16) return fail(G4_EINVAL, "%s: x_type %u (f32, f16 or bf16)", what, p->x_type);
    if (p->reserved) return fail(G4_EINVAL, "%s: reserved must be 0", what);
    if (!x || !out || !scales) return fail(G4_EINVAL, "%s: NULL x, out or scales", what);
    NormRowsArgs a = {};
    a.x_stride = p->x_stride;
    a.out_stride = p->out_stride;
    if ((rc = stride_check(what, "x", a.x_stride, p->n)) || (rc = stride_check(what, "out", a.out_stride, p->n))) return rc;
    if ((rc = pointer_check(what, "x", x, p->x_type)) || (rc = pointer_check(what, "scales", scales, G4_F32))) return rc;
    if (out == x) return fail(G4_EINVAL, "%s: out is x", what);
    if (p->rows == 0) return G4_OK;
    const Operand o_x = rows_operand("x", x, p->x_type, p->n, a.x_stride, p->rows),
                  o_out = rows_operand("out", out, G4_E4M3, p->n, a.out_stride, p->rows),
                  o_scales = {"scales", one_range(scales, 4ull * p->rows)};
    if ((rc = apart_check(what, o_out, {o_x, o_scales})) || (rc = apart_check(what, o_scales, {o_x}))) return rc;
    a.x = x;
    a.out = out;
    a.scales = scales;
    a.rows = p->rows;
    a.n = p->n;
    a.x_type = p->x_type;
    a.out_type = G4_E4M3;
    const bool wide = p->n % 8 == 0 && wide_rows(x, a.x_type, a.x_stride) && wide_rows(out, G4_E4M3, a.out_stride);
    launch_norm_rows(a, wide, as_stream(stream));
    G4_CHECK_LAUNCH("k_norm_rows");
    return G4_OK;
}

}  // extern "C"
