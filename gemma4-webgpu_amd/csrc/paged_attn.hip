// Attention of a batch's new tokens (single ones, chains, trees of drafted
// tokens) over a paged cache: g4_paged_attn.
//
// Per query row r = (token, query head of a kv head) and attended cache row i:
//   s_i = scale q.k_i (capped: softcap tanh(s / softcap)), p_i = e^(s_i - m),
//   out = sum p_i v_i / sum p_i, with the running maximum m and sum of an online
//   softmax, f32 throughout; K and V are read once per tile of 16 C query rows.
//
// MFMA mapping (v_mfma_f32_16x16x32_f16; lane = 16 g + n), for each 32-row tile of
// the cache, per group of 16 query rows:
//   S^T[16 rows x 16 q] = K[16 x 32 d] Q^T: lane (n, g) supplies 8 elements of K row n,
//     straight from the cache; the query is f16, so products are exact.
//   O^T[16 d x 16 q] += V^T[16 d x 32 rows] P^T: lane (n, g) holds V pieces of rows
//     4g..4g+3 and 16+4g..16+4g+3, the rows whose scores it has, and transposes them in
//     registers. P goes in twice, as its f16 value and the f16 residual: 22 bits, so that
//     an f32 result keeps f32 accuracy (one f16 P alone leaves 2e-4).
// e4m3 pools are widened to f16 in registers, which is exact.
//
// Work split: a (sequence, kv head, tile of query rows) is an item of ceil(rows / 32)
// row tiles; all items' tiles in order are cut into equal shares, one a workgroup,
// whatever the lengths, so a ragged batch fills the chip and one long sequence does
// too. Lengths are read on the device (a captured launch serves the next step's),
// every workgroup finds its share by a scan over the sequences. An item cut between
// workgroups leaves (m, l, o) records that a second launch joins in a fixed order.
#include "decode_core.h"
#include "paged.h"

namespace g4 {

constexpr int kPagedWaves = 4;
constexpr int kPagedThreads = 64 * kPagedWaves;

struct PagedAttnArgs {
    const uint16_t* __restrict__ q;
    float* __restrict__ out;
    const char* __restrict__ k;
    const char* __restrict__ v;
    float* __restrict__ part_o;   // [2 * workgroups][16 C][HD]
    float* __restrict__ part_ml;  // [2 * workgroups][16 C][2]
    uint32_t nkh, group;
    int32_t window;               // 0: none
    float scale, cap, inv_cap;
    uint32_t wgs, min_share;      // workgroups of the attention launch; least tiles a workgroup takes
    PagedBatchDev b;
};

// ---- the items ----------------------------------------------------------------

// Row tiles of query tile qt (16 C rows) of a sequence: [first, first + n), n >= 1.
// hi: one past the last row that any of its tokens attends.
struct PagedSpan {
    unsigned first, n, hi;
};
template <int C>
__device__ __forceinline__ PagedSpan paged_span(const PagedAttnArgs& a, const PagedSeq& sq, unsigned qt) {
    const unsigned j0 = qt * (16 * C) / a.group;
    const unsigned j1 = min((qt * (16 * C) + 16 * C - 1) / a.group, sq.n - 1);
    const unsigned hi = min(sq.ctx + (a.b.mask ? sq.n : j1 + 1), paged_rows(a.b));
    unsigned lo = 0;
    if (a.window) {  // positions are at least ctx (a chain's: ctx + j)
        const int at = (int)(sq.ctx + (a.b.positions || a.b.mask ? 0u : j0)) - a.window + 1;
        lo = min((unsigned)max(at, 0), sq.ctx);
    }
    lo = min(lo, hi - 1);
    PagedSpan s;
    s.first = lo / 32;
    s.n = (hi + 31) / 32 - s.first;
    s.hi = hi;
    return s;
}
template <int C>
__device__ __forceinline__ unsigned paged_q_tiles(const PagedAttnArgs& a, const PagedSeq& sq) {
    return (sq.n * a.group + 16 * C - 1) / (16 * C);
}
// Row tiles of all query tiles of one kv head of a sequence.
template <int C>
__device__ __forceinline__ unsigned paged_tiles(const PagedAttnArgs& a, const PagedSeq& sq) {
    unsigned u = 0;
    const unsigned nq = paged_q_tiles<C>(a, sq);
    for (unsigned qt = 0; qt < nq; qt++) u += paged_span<C>(a, sq, qt).n;
    return u;
}

__device__ __forceinline__ unsigned wave_scan(unsigned x, unsigned lane) {  // inclusive
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const unsigned y = __shfl_up(x, d);
        if (lane >= (unsigned)d) x += y;
    }
    return x;
}
__device__ __forceinline__ unsigned lane_value(unsigned x, unsigned lane) {
    return __builtin_amdgcn_readlane(x, lane);
}

// The batch's row tiles, as a wave sees them: lane l holds sequence l of a group of 64.
template <int C>
struct PagedScan {
    unsigned total = 0;           // row tiles of the whole batch
    unsigned tiles = 0, incl = 0;  // of the group held: a sequence's (all kv heads), and up to it

    __device__ __forceinline__ void group(const PagedAttnArgs& a, unsigned s0, unsigned lane) {
        const unsigned s = s0 + lane;
        tiles = 0;
        if (s < a.b.n_seqs) tiles = paged_tiles<C>(a, paged_seq(a.b, s)) * a.nkh;
        incl = wave_scan(tiles, lane);
    }
    __device__ __forceinline__ void run(const PagedAttnArgs& a, unsigned lane) {
        for (unsigned s0 = 0; s0 < a.b.n_seqs; s0 += 64) {
            group(a, s0, lane);
            total += lane_value(incl, 63);
        }
    }
    // Tiles a workgroup takes (the last one fewer).
    __device__ __forceinline__ unsigned share(const PagedAttnArgs& a) const {
        return max((total + a.wgs - 1) / a.wgs, a.min_share);
    }
};

// An item and where a tile number lies in it.
struct PagedPlace {
    unsigned s, kvh, qt;
    unsigned off;   // tiles of the item before it
    unsigned base;  // the item's first tile number
};
template <int C>
__device__ __forceinline__ PagedPlace paged_place(const PagedAttnArgs& a, PagedScan<C>& scan, unsigned u, unsigned lane) {
    PagedPlace p{};
    unsigned before = 0;
    for (unsigned s0 = 0;; s0 += 64) {
        if (a.b.n_seqs > 64) scan.group(a, s0, lane);
        const unsigned all = lane_value(scan.incl, 63);
        if (u < before + all || s0 + 64 >= a.b.n_seqs) {
            const unsigned l = __builtin_ctzll(__ballot(scan.incl > u - before) | (1ull << 63));
            p.s = s0 + l;
            before += lane_value(scan.incl, l) - lane_value(scan.tiles, l);
            const unsigned per_head = lane_value(scan.tiles, l) / a.nkh;
            const unsigned rem = u - before;
            p.kvh = rem / per_head;
            p.off = rem % per_head;
            p.base = before + p.kvh * per_head;
            break;
        }
        before += all;
    }
    const PagedSeq sq = paged_seq(a.b, p.s);
    for (;;) {
        const unsigned n = paged_span<C>(a, sq, p.qt).n;
        if (p.off < n) break;
        p.off -= n;
        p.base += n;
        p.qt++;
    }
    return p;
}

// ---- cache tiles ----------------------------------------------------------------

template <int HD, bool F8>
struct PagedDims {
    static constexpr int ES = F8 ? 1 : 2;           // bytes an element
    static constexpr int NC = HD / 32;              // score MFMAs a 16-row half (32 d each)
    static constexpr int KP = HD * ES / 64;         // 16-byte K pieces a lane (4 lanes a row: 64 bytes)
    static constexpr int VP = HD * ES / 256;        // V pieces a lane and row (16 lanes a row: 256 bytes)
    static constexpr int E = 16 / ES;               // elements a piece
    static constexpr int NO = HD / 16;              // output MFMA tiles of 16 d
};

// A lane's V pieces of a tile: [piece block][row].
template <int HD, bool F8>
using PagedV = u32x4[PagedDims<HD, F8>::VP][8];

__device__ __forceinline__ uint32_t fp8x2_f16(uint32_t w, bool high) {
    return high ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true))
                : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
}

// Elements of chunk c of the score product for lane group g: f16 32 c + 8 g .. + 8; e4m3
// pieces hold two chunks' elements, 64 (c / 2) + 16 g + 8 (c % 2) .. + 8.
template <bool F8>
__device__ __forceinline__ int paged_q_elem(int c, int g) {
    return F8 ? 64 * (c >> 1) + 16 * g + 8 * (c & 1) : 32 * c + 8 * g;
}
template <int HD, bool F8>
__device__ __forceinline__ f16x8 paged_k_chunk(const u32x4 (&kr)[PagedDims<HD, F8>::KP], int c) {
    if constexpr (F8) {
        const uint32_t a = kr[c >> 1][2 * (c & 1)], b = kr[c >> 1][2 * (c & 1) + 1];
        return __builtin_bit_cast(f16x8, u32x4{fp8x2_f16(a, false), fp8x2_f16(a, true), fp8x2_f16(b, false), fp8x2_f16(b, true)});
    } else {
        return __builtin_bit_cast(f16x8, kr[c]);
    }
}

// 16 rows of K from a wave-uniform address: lane (n, g) pieces of row n.
template <int HD, bool F8>
__device__ __forceinline__ void paged_load_k(const char* base, uint32_t row_bytes, int n, int g,
                                             u32x4 (&kr)[PagedDims<HD, F8>::KP]) {
    const uint32_t off = (uint32_t)n * row_bytes + (uint32_t)g * 16u;
#pragma unroll
    for (int c = 0; c < PagedDims<HD, F8>::KP; c++) kr[c] = ldg<u32x4>(base + (off + c * 64u));
}
// The two 16-row halves of V: lane (n, g) piece n of rows 4g + t of either half (t < 4: the first).
template <int HD, bool F8>
__device__ __forceinline__ void paged_load_v(const char* base0, const char* base1, uint32_t row_bytes, int n, int g,
                                             PagedV<HD, F8>& vr) {
    const uint32_t off = (uint32_t)(4 * g) * row_bytes + (uint32_t)n * 16u;
#pragma unroll
    for (int t = 0; t < 8; t++)
#pragma unroll
        for (int b = 0; b < PagedDims<HD, F8>::VP; b++)
            vr[b][t] = ldg<u32x4>((t < 4 ? base0 : base1) + (off + (uint32_t)(t & 3) * row_bytes + b * 256u));
}

// tanh(x) to f32 accuracy (logprobs.hip has the derivation).
__device__ __forceinline__ float paged_tanh(float x) {
    const float ax = fabsf(x), z = x * x;
    const float t = __builtin_amdgcn_exp2f(-2.0f * kLog2e * ax);
    const bool small = ax < 0.5f;
    const float num = small ? ax * (945.0f + z * (105.0f + z)) : 1.0f - t;
    const float den = small ? 945.0f + z * (420.0f + 15.0f * z) : 1.0f + t;
    const float y = __builtin_amdgcn_rcpf(den), q = num * y;
    return copysignf(__builtin_fmaf(__builtin_fmaf(-q, den, num), y, q), x);
}

// O^T += V^T P^T for one piece block, all query groups. Word w of a row's piece holds
// elements (2w, 2w + 1) (f16) or 4w .. 4w + 3 (e4m3): acc tile b E + e takes element e of
// every lane's piece, so its rows are d = 16 E b + E (row) + e.
template <int HD, int C, bool F8>
__device__ __forceinline__ void paged_pv(const PagedV<HD, F8>& vr, const f16x8 (&hi)[C],
                                         const f16x8 (&lo)[C], f32x4 (&acc)[C][PagedDims<HD, F8>::NO]) {
    using D = PagedDims<HD, F8>;
#pragma unroll
    for (int b = 0; b < D::VP; b++)
#pragma unroll
        for (int w = 0; w < 4; w++)
#pragma unroll
            for (int h = 0; h < (F8 ? 2 : 1); h++) {
                uint32_t x[8];
#pragma unroll
                for (int t = 0; t < 8; t++) x[t] = F8 ? fp8x2_f16(vr[b][t][w], h) : vr[b][t][w];
                u32x4 e0, e1;
#pragma unroll
                for (int p = 0; p < 4; p++) {
                    e0[p] = perm_lo(x[2 * p], x[2 * p + 1]);
                    e1[p] = perm_hi(x[2 * p], x[2 * p + 1]);
                }
                const int i = b * D::E + (F8 ? 4 * w + 2 * h : 2 * w);
#pragma unroll
                for (int c = 0; c < C; c++) {
                    acc[c][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, e0), hi[c], acc[c][i], 0, 0, 0);
                    acc[c][i + 1] =
                        __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, e1), hi[c], acc[c][i + 1], 0, 0, 0);
                }
#pragma unroll
                for (int c = 0; c < C; c++) {
                    acc[c][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, e0), lo[c], acc[c][i], 0, 0, 0);
                    acc[c][i + 1] =
                        __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, e1), lo[c], acc[c][i + 1], 0, 0, 0);
                }
                if constexpr (HD == 512) __builtin_amdgcn_sched_barrier(0);
            }
}

// Words of V pieces whose elements are Inf or NaN (exponent all ones; e4m3: NaN alone): their places, as
// the elements' top bits.
template <bool F8>
__device__ __forceinline__ uint32_t odd_elements(uint32_t w) {
    return F8 ? ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u : ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
}

// Takes Inf and NaN out of a lane's V pieces; returns the rows (bit t) that had some.
template <int HD, bool F8>
__device__ __forceinline__ unsigned paged_take_odd(PagedV<HD, F8>& vr) {
    unsigned rows = 0;
#pragma unroll
    for (int t = 0; t < 8; t++) {
        uint32_t any = 0;
#pragma unroll
        for (int b = 0; b < PagedDims<HD, F8>::VP; b++)
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const uint32_t odd = odd_elements<F8>(vr[b][t][w]);
                any |= odd;
                const uint32_t low = odd >> (F8 ? 7 : 15);  // each odd element's bit 0, times all ones
                vr[b][t][w] &= ~(low * (F8 ? 0xffu : 0xffffu));
            }
        rows |= (any ? 1u : 0u) << t;
    }
    return rows;
}

// What one V row's Inf and NaN elements give the outputs of a lane whose column attends the row.
template <int HD, bool F8>
__device__ __forceinline__ void paged_add_odd(const char* row, int g, bool attends, f32x4 (&acc)[PagedDims<HD, F8>::NO]) {
    using D = PagedDims<HD, F8>;
#pragma unroll
    for (int i = 0; i < D::NO; i++) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int d = 16 * D::E * (i / D::E) + D::E * (4 * g + j) + i % D::E;
            float x;
            if constexpr (F8) x = (ldg<uint8_t>(row + d) & 0x7f) == 0x7f ? __uint_as_float(0x7FC00000u) : 0.0f;
            else x = h2f(ldg<uint16_t>(row + 2 * d));
            if (attends && !(fabsf(x) < INFINITY)) acc[i][j] += x;
        }
        __builtin_amdgcn_sched_barrier(0);  // tile by tile: the registers hold no more
    }
}

// ---- attention --------------------------------------------------------------------

template <int HD, int C>
struct PagedSmem {
    f16x8 q[C][HD / 32][64];                           // score operand, lane-major
    float o[kPagedWaves][HD / 16 * 4][64];             // one query group's outputs, per wave
    float m[kPagedWaves][16 * C], l[kPagedWaves][16 * C];
};

template <int HD, int C, bool F8>
__global__ __launch_bounds__(kPagedThreads, C == 1 && HD == 256 ? 2 : 1) void k_paged_attn(const PagedAttnArgs a) {
    using D = PagedDims<HD, F8>;
    __shared__ PagedSmem<HD, C> sm;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, g = lane >> 4;
    const unsigned G = a.group;

    PagedScan<C> scan;
    scan.run(a, lane);
    const unsigned share = scan.share(a);
    const uint64_t first = (uint64_t)blockIdx.x * share;
    if (first >= scan.total) return;  // uniform
    unsigned u = (unsigned)first;
    const unsigned u_end = min(u + share, scan.total);
    PagedPlace at = paged_place<C>(a, scan, u, lane);
    const uint32_t row_bytes = a.nkh * HD * D::ES;
    const unsigned page_rows = 1u << a.b.page_shift;

    while (u < u_end) {  // one item or a part of one
        const unsigned s = __builtin_amdgcn_readfirstlane(at.s);
        const PagedSeq sq = paged_seq(a.b, s);
        const unsigned kvh = __builtin_amdgcn_readfirstlane(at.kvh), qt = __builtin_amdgcn_readfirstlane(at.qt);
        const PagedSpan sp = paged_span<C>(a, sq, qt);
        const unsigned off = __builtin_amdgcn_readfirstlane(at.off);
        const unsigned seg = min(sp.n - off, u_end - u);
        const unsigned rows = sq.n * G;               // query rows of this (sequence, kv head)
        const uint64_t head_off = (uint64_t)kvh * HD * D::ES;
        const int32_t* table = a.b.table + (uint64_t)s * a.b.table_stride;

        // The query tile into LDS: column n of group c is query row 16 (C qt + c) + n.
        __syncthreads();  // the last segment's combine has read sm
        for (int i = threadIdx.x; i < C * D::NC * 64; i += kPagedThreads) {
            const int l = i & 63, c = i / 64 % D::NC, cg = i / 64 / D::NC;
            const unsigned r = (qt * C + cg) * 16 + (l & 15);
            f16x8 x = {};
            if (r < rows) {
                const unsigned tok = sq.start + r / G;
                x = ldg<f16x8>(a.q + ((uint64_t)tok * (a.nkh * G) + kvh * G + r % G) * HD + paged_q_elem<F8>(c, l >> 4));
            }
            sm.q[cg][c][l] = x;
        }
        // The lane's columns.
        unsigned jq[C];  // new-token index, or ~0 past the rows
        int pos[C];
        uint64_t bits[C];
#pragma unroll
        for (int c = 0; c < C; c++) {
            const unsigned r = (qt * C + c) * 16 + n;
            jq[c] = r < rows ? r / G : ~0u;
            const unsigned tok = sq.start + (r < rows ? r / G : 0u);
            pos[c] = a.b.positions ? max(a.b.positions[tok], 0) : (int)(sq.ctx + (r < rows ? r / G : 0u));
            bits[c] = a.b.mask ? a.b.mask[(uint64_t)tok * a.b.mask_words] : 0;
        }
        __syncthreads();

        float m_run[C], l_run[C];
        f32x4 acc[C][D::NO];
#pragma unroll
        for (int c = 0; c < C; c++) {
            m_run[c] = -INFINITY;
            l_run[c] = 0.0f;
#pragma unroll
            for (int i = 0; i < D::NO; i++) acc[c][i] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        // Rows that every column attends: committed, and above every window's start.
        const unsigned clear_hi = sq.ctx;
        unsigned clear_lo = 0;
        if (a.window)
            clear_lo = a.b.positions ? sq.ctx : (unsigned)max((int)(sq.ctx + sq.n) - a.window, 0);

        unsigned pages0 = 0, pages1 = 0;  // lane i: page of the two 16-row halves of the wave's tile i (of 64)
        unsigned have = 0;
        for (unsigned it = 0, t = wave; t < seg; it++, t += kPagedWaves) {
            if (it == have) {  // uniform
                const unsigned r0 = (sp.first + off + wave + kPagedWaves * (it + lane)) * 32;
                const unsigned p0 = min(r0, sp.hi - 1) >> a.b.page_shift, p1 = min(r0 + 16, sp.hi - 1) >> a.b.page_shift;
                pages0 = (unsigned)table[p0];
                pages1 = (unsigned)table[p1];
                have += 64;
            }
            const unsigned kt0 = (sp.first + off + t) * 32;
            const unsigned pg0 = lane_value(pages0, it & 63), pg1 = lane_value(pages1, it & 63);
            const bool ok0 = pg0 < a.b.num_pages, ok1 = pg1 < a.b.num_pages;
            const unsigned in0 = kt0 & (page_rows - 1), in1 = (kt0 + 16) & (page_rows - 1);
            const uint64_t at0 = (((uint64_t)(ok0 ? pg0 : 0u) << a.b.page_shift) + in0) * row_bytes + head_off;
            const uint64_t at1 = (((uint64_t)(ok1 ? pg1 : 0u) << a.b.page_shift) + in1) * row_bytes + head_off;
            u32x4 kr[2][D::KP];
            u32x4 vr[D::VP][8];
            paged_load_k<HD, F8>(a.k + at0, row_bytes, n, g, kr[0]);
            paged_load_k<HD, F8>(a.k + at1, row_bytes, n, g, kr[1]);
            paged_load_v<HD, F8>(a.v + at0, a.v + at1, row_bytes, n, g, vr);

            f32x4 sc[C][2];
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int h = 0; h < 2; h++) sc[c][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ch = 0; ch < D::NC; ch++) {
                const f16x8 k0 = paged_k_chunk<HD, F8>(kr[0], ch), k1 = paged_k_chunk<HD, F8>(kr[1], ch);
#pragma unroll
                for (int c = 0; c < C; c++) {
                    const f16x8 qv = sm.q[c][ch][lane];
                    sc[c][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qv, sc[c][0], 0, 0, 0);
                    sc[c][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qv, sc[c][1], 0, 0, 0);
                }
            }
            const bool clear = kt0 >= clear_lo && kt0 + 32 <= clear_hi && ok0 && ok1;
            unsigned seen[C];  // bit t: column c of this lane attends the lane's row t
#pragma unroll
            for (int c = 0; c < C; c++) seen[c] = 0xffu;
            if (!clear) {
#pragma unroll
                for (int c = 0; c < C; c++) seen[c] = 0;
                unsigned dead = 0;
                for (int t8 = 0; t8 < 8; t8++) {
                    const unsigned row = kt0 + (t8 < 4 ? 0 : 16) + 4 * g + (t8 & 3);
                    if (row >= sp.hi || !(t8 < 4 ? ok0 : ok1)) {
                        dead |= 1u << t8;
                        continue;
                    }
                    const unsigned dj = row - sq.ctx;  // new-token index (row >= ctx)
                    int rpos = (int)row;
                    if (row >= sq.ctx && a.window && a.b.positions) rpos = max(a.b.positions[sq.start + dj], 0);
#pragma unroll
                    for (int c = 0; c < C; c++) {
                        bool ok = jq[c] != ~0u;
                        if (row >= sq.ctx) {
                            if (a.b.mask) {
                                uint64_t word = bits[c];
                                if (a.b.mask_words > 1 && ok)
                                    word = a.b.mask[(uint64_t)(sq.start + jq[c]) * a.b.mask_words + (dj >> 6)];
                                ok = ok && ((word >> (dj & 63)) & 1);
                            } else {
                                ok = ok && dj <= jq[c];
                            }
                        }
                        if (a.window) ok = ok && rpos > pos[c] - a.window;
                        seen[c] |= (ok ? 1u : 0u) << t8;
                    }
                }
#pragma unroll
                for (int t8 = 0; t8 < 8; t8++)
                    if (dead >> t8 & 1) {
#pragma unroll
                        for (int b = 0; b < D::VP; b++) vr[b][t8] = u32x4{0u, 0u, 0u, 0u};
                    }
            }
            f16x8 hi[C], lo[C];
#pragma unroll
            for (int c = 0; c < C; c++) {
                float sv[8];
                float tmax = -INFINITY;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    float x = sc[c][i >> 2][i & 3] * a.scale;
                    if (a.cap > 0.0f) x = a.cap * paged_tanh(x * a.inv_cap);
                    sv[i] = seen[c] >> i & 1 ? x : -INFINITY;
                    tmax = fmaxf(tmax, sv[i]);
                }
                tmax = max_xor16(tmax);  // the column's rows lie in four lane groups
                tmax = max_xor32(tmax);
                const float m_new = fmaxf(m_run[c], tmax);
                if (__any(m_new > m_run[c])) {
                    const float alpha = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m_run[c] - m_new) * kLog2e);
                    l_run[c] *= alpha;
#pragma unroll
                    for (int i = 0; i < D::NO; i++) acc[c][i] *= alpha;
                }
                m_run[c] = m_new;
                const float base = m_new == -INFINITY ? 0.0f : m_new;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float p = __builtin_amdgcn_exp2f((sv[i] - base) * kLog2e);
                    l_run[c] += p;
                    const f16 h = (f16)p;
                    hi[c][i] = h;
                    lo[c][i] = (f16)(p - (float)h);
                }
            }
            // Rows that only some columns attend may hold Inf or NaN, and 0 times those is no 0: they are
            // left out of the products and added to the columns that attend them.
            uint32_t odd_rows = 0;  // bit 4 t + g: the row t of lane group g; uniform
            if (!clear) {
                unsigned odd = 0;
#pragma unroll
                for (int b = 0; b < D::VP; b++)
#pragma unroll
                    for (int t8 = 0; t8 < 8; t8++)
#pragma unroll
                        for (int w = 0; w < 4; w++) odd |= odd_elements<F8>(vr[b][t8][w]);
                if (__any(odd != 0)) {
                    const unsigned mine = paged_take_odd<HD, F8>(vr);
                    for (int t8 = 0; t8 < 8; t8++) {
                        const uint64_t b = __ballot(mine >> t8 & 1);
                        for (int gg = 0; gg < 4; gg++) odd_rows |= (b >> (16 * gg) & 0xffff ? 1u : 0u) << (4 * t8 + gg);
                    }
                }
            }
            paged_pv<HD, C, F8>(vr, hi, lo, acc);
            while (odd_rows) {
                const int bit = __builtin_ctz(odd_rows), t8 = bit >> 2, gg = bit & 3;
                odd_rows &= odd_rows - 1;
                const char* row = a.v + (t8 < 4 ? at0 : at1) + (uint32_t)(4 * gg + (t8 & 3)) * row_bytes;
#pragma unroll
                for (int c = 0; c < C; c++)
                    paged_add_odd<HD, F8>(row, g, __shfl(seen[c], 16 * gg + n) >> t8 & 1, acc[c]);
            }
        }

        // The four waves' states joined: maxima first, then a query group's outputs at a time.
        const bool whole = seg == sp.n;
        const unsigned slot = 2 * blockIdx.x + (off ? 0u : 1u);  // a part that begins its item, or continues one
#pragma unroll
        for (int c = 0; c < C; c++) {
            float l = add_xor16(l_run[c]);
            l = add_xor32(l);
            if (g == 0) {
                sm.m[wave][16 * c + n] = m_run[c];
                sm.l[wave][16 * c + n] = l;
            }
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < C; c++) {
            float M = -INFINITY, L = 0.0f;
#pragma unroll
            for (int w = 0; w < kPagedWaves; w++) M = fmaxf(M, sm.m[w][16 * c + n]);
            const float base = M == -INFINITY ? 0.0f : M;
#pragma unroll
            for (int w = 0; w < kPagedWaves; w++)
                L += sm.l[w][16 * c + n] * __builtin_amdgcn_exp2f((sm.m[w][16 * c + n] - base) * kLog2e);
            const float f = __builtin_amdgcn_exp2f((m_run[c] - base) * kLog2e);
#pragma unroll
            for (int i = 0; i < D::NO; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) sm.o[wave][i * 4 + j][lane] = acc[c][i][j] * f;
            __syncthreads();
            const unsigned r = (qt * C + c) * 16 + n;
            if (r < rows) {
                const float inv = whole ? (L > 0.0f ? 1.0f / L : (L == 0.0f ? 0.0f : L)) : 1.0f;
                float* dst = whole ? a.out + ((uint64_t)(sq.start + r / G) * (a.nkh * G) + kvh * G + r % G) * HD
                                   : a.part_o + ((uint64_t)slot * (16 * C) + 16 * c + n) * HD;
                if (!whole && wave == 0 && g == 0)
                    stg<f32x2>(a.part_ml + ((uint64_t)slot * (16 * C) + 16 * c + n) * 2, f32x2{M, L});
                const int j = wave;  // of the 4 rows 4g + j of every output tile
#pragma unroll
                for (int b = 0; b < D::VP; b++) {
                    const int d0 = 16 * D::E * b + D::E * (4 * g + j);
#pragma unroll
                    for (int e = 0; e < D::E; e += 4) {
                        f32x4 x;
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int k = (b * D::E + e + i) * 4 + j;
                            x[i] = ((sm.o[0][k][lane] + sm.o[1][k][lane]) + (sm.o[2][k][lane] + sm.o[3][k][lane])) * inv;
                        }
                        stg<f32x4>(dst + d0 + e, x);
                    }
                }
            }
            __syncthreads();
        }

        u += seg;
        at.off = 0;
        if (u < u_end) {  // the next item: this head's next query tile, the next head, the next sequence with tokens
            at.qt = qt + 1;
            at.kvh = kvh;
            at.s = s;
            if (at.qt >= paged_q_tiles<C>(a, sq)) {
                at.qt = 0;
                at.kvh++;
                if (at.kvh >= a.nkh) {
                    at.kvh = 0;
                    do at.s++;
                    while (at.s < a.b.n_seqs && paged_seq(a.b, at.s).n == 0);
                }
            }
        }
    }
}

// ---- the join ------------------------------------------------------------------------

// Workgroup (item, rows): the records of an item that was cut, in the order of its
// rows. HD / 4 threads a query row. Items beyond the batch's and items that one
// workgroup had leave at once.
template <int HD, int C>
__global__ __launch_bounds__(256) void k_paged_join(const PagedAttnArgs a, uint32_t per_seq) {
    constexpr unsigned TPR = HD / 4, R = 256 / TPR;
    const unsigned lane = threadIdx.x & 63;
    const unsigned per_head = per_seq / a.nkh;  // query tiles of a kv head at most
    const unsigned s = blockIdx.x / per_seq, kvh = blockIdx.x % per_seq / per_head, qt = blockIdx.x % per_head;
    const PagedSeq sq = paged_seq(a.b, s);
    if (sq.n == 0 || qt >= paged_q_tiles<C>(a, sq)) return;  // uniform
    // The item's first tile number, and the share.
    PagedScan<C> scan;
    unsigned base = 0;
    for (unsigned s0 = 0; s0 < a.b.n_seqs; s0 += 64) {
        scan.group(a, s0, lane);
        if (s >= s0 && s < s0 + 64) base = scan.total + lane_value(scan.incl, s - s0) - lane_value(scan.tiles, s - s0);
        scan.total += lane_value(scan.incl, 63);
    }
    const unsigned share = scan.share(a);
    unsigned head = 0, mine = 0;
    const unsigned nq = paged_q_tiles<C>(a, sq);
    for (unsigned i = 0; i < nq; i++) {
        const unsigned t = paged_span<C>(a, sq, i).n;
        if (i < qt) base += t;
        if (i == qt) mine = t;
        head += t;
    }
    base += kvh * head;
    const unsigned w0 = base / share, w1 = (base + mine - 1) / share;
    if (w0 == w1) return;  // uniform: one workgroup wrote the result
    const unsigned r16 = blockIdx.y * R + threadIdx.x / TPR, r = qt * (16 * C) + r16;
    if (r >= sq.n * a.group) return;
    const unsigned d = threadIdx.x % TPR * 4;
    // The first record is its workgroup's slot 1, the others continue the item: slot 0.
    auto rec = [&](unsigned w) __attribute__((always_inline)) { return ((uint64_t)2 * w + (w == w0 ? 1u : 0u)) * (16 * C) + r16; };
    float M = -INFINITY;
    for (unsigned w = w0; w <= w1; w++) M = fmaxf(M, ldg<f32x2>(a.part_ml + rec(w) * 2)[0]);
    const float ref = M == -INFINITY ? 0.0f : M;
    float L = 0.0f;
    f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
    for (unsigned w = w0; w <= w1; w++) {
        const f32x2 ml = ldg<f32x2>(a.part_ml + rec(w) * 2);
        const float f = __builtin_amdgcn_exp2f((ml[0] - ref) * kLog2e);
        const f32x4 x = ldg<f32x4>(a.part_o + rec(w) * HD + d);
        L += ml[1] * f;
        o += x * f;
    }
    const float inv = L > 0.0f ? 1.0f / L : (L == 0.0f ? 0.0f : L);
    stg<f32x4>(a.out + ((uint64_t)(sq.start + r / a.group) * (a.nkh * a.group) + kvh * a.group + r % a.group) * HD + d, o * inv);
}

// ---- host --------------------------------------------------------------------------

struct PagedPlan {
    unsigned c, wgs;
    uint64_t q_tiles;  // of a kv head, at most
    size_t bytes;
};
static PagedPlan paged_plan(unsigned head_dim, unsigned num_kv_heads, unsigned num_q_heads, const PagedBatchDev& b) {
    PagedPlan p;
    const uint64_t rows = (uint64_t)b.max_tokens * (num_q_heads / num_kv_heads);
    p.c = 1;
    p.q_tiles = (rows + 16 * p.c - 1) / (16 * p.c);
    p.wgs = device_cus() * (p.c == 1 && head_dim == 256 ? 2 : 1);
    p.bytes = (size_t)2 * p.wgs * 16 * p.c * (head_dim + 2) * sizeof(float);
    return p;
}

template <int HD, int C, bool F8>
static void launch_paged(const PagedAttnArgs& a, const PagedPlan& p, hipStream_t st) {
    G4_LAUNCH((k_paged_attn<HD, C, F8>), dim3(p.wgs), dim3(kPagedThreads), 0, st, a);
    const uint32_t per_seq = (uint32_t)p.q_tiles * a.nkh;
    G4_LAUNCH((k_paged_join<HD, C>), dim3(a.b.n_seqs * per_seq, 16 * C * HD / 4 / 256), dim3(256), 0, st, a, per_seq);
}

}  // namespace g4

using namespace g4;

namespace {

int paged_attn_check(const g4_paged_cache* cache, const g4_paged_batch* batch, uint32_t num_q_heads, PagedBatchDev* b) {
    const int rc = paged_check("pagedAttn", cache, batch, b);
    if (rc) return rc;
    if (num_q_heads == 0 || num_q_heads % cache->num_kv_heads || num_q_heads / cache->num_kv_heads > (uint32_t)kMaxGroup)
        return fail(G4_EINVAL, "pagedAttn: %u query heads over %u kv heads (a multiple, up to %d times)", num_q_heads,
                    cache->num_kv_heads, kMaxGroup);
    const PagedPlan p = paged_plan(cache->head_dim, cache->num_kv_heads, num_q_heads, *b);
    const uint64_t items = (uint64_t)b->n_seqs * cache->num_kv_heads * p.q_tiles;
    const uint64_t tiles = ((uint64_t)b->table_stride * cache->page_size + 31) / 32;
    if (items > (1u << 23) || items * tiles > 0x7fffffffull)
        return fail(G4_EINVAL, "pagedAttn: %u sequences of up to %u tokens over %u pages are too much for one call",
                    b->n_seqs, b->max_tokens, b->table_stride);
    return G4_OK;
}

}  // namespace

extern "C" {

int g4_paged_attn_workspace_size(const g4_paged_cache* cache, const g4_paged_batch* batch, uint32_t num_q_heads,
                                 size_t* bytes) {
    if (!bytes) return fail(G4_EINVAL, "g4_paged_attn_workspace_size: bytes is NULL");
    PagedBatchDev b = {};
    const int rc = paged_attn_check(cache, batch, num_q_heads, &b);
    if (rc) return rc;
    *bytes = paged_plan(cache->head_dim, cache->num_kv_heads, num_q_heads, b).bytes;
    return G4_OK;
}

int g4_paged_attn(const g4_paged_cache* cache, const g4_paged_batch* batch, const uint16_t* q, float* out,
                  const g4_paged_attn_params* p, void* workspace, size_t workspace_bytes, void* stream) {
    if (!p) return fail(G4_EINVAL, "pagedAttn: NULL params");
    PagedAttnArgs a = {};
    const int rc = paged_attn_check(cache, batch, p->num_q_heads, &a.b);
    if (rc) return rc;
    if (!q || !out || !workspace) return fail(G4_EINVAL, "pagedAttn: NULL q, out or workspace");
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15)
        return fail(G4_EINVAL, "pagedAttn: q, out and workspace must be 16-byte aligned");
    if (!(p->scale > -1e30f && p->scale < 1e30f)) return fail(G4_EINVAL, "pagedAttn: scale %g", (double)p->scale);
    if (!(p->softcap >= 0.0f) || p->softcap > 1e30f || (p->softcap > 0.0f && p->softcap < 1e-6f))
        return fail(G4_EINVAL, "pagedAttn: softcap %g (0, or 1e-6 to 1e30)", (double)p->softcap);
    const PagedPlan plan = paged_plan(cache->head_dim, cache->num_kv_heads, p->num_q_heads, a.b);
    if (workspace_bytes < plan.bytes)
        return fail(G4_ENOSPC, "pagedAttn: workspace %zu bytes < %zu needed", workspace_bytes, plan.bytes);
    if (batch->n_tokens == 0) return G4_OK;
    a.q = q;
    a.out = out;
    a.k = static_cast<const char*>(cache->k_pool);
    a.v = static_cast<const char*>(cache->v_pool);
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + (size_t)2 * plan.wgs * 16 * plan.c * cache->head_dim;
    a.nkh = cache->num_kv_heads;
    a.group = p->num_q_heads / cache->num_kv_heads;
    a.window = p->sliding_window > (1u << 30) ? 0 : (int32_t)p->sliding_window;  // positions are below 2^31 - 2^30
    a.scale = p->scale;
    a.cap = p->softcap;
    a.inv_cap = p->softcap > 0.0f ? 1.0f / p->softcap : 0.0f;
    a.wgs = plan.wgs;
    a.min_share = 8;
    hipStream_t st = as_stream(stream);
    const bool f8 = cache->dtype == G4_KV_E4M3;
    if (cache->head_dim == 512) {
        if (f8) launch_paged<512, 1, true>(a, plan, st);
        else launch_paged<512, 1, false>(a, plan, st);
    } else {
        if (f8) launch_paged<256, 1, true>(a, plan, st);
        else launch_paged<256, 1, false>(a, plan, st);
    }
    G4_CHECK_LAUNCH("pagedAttn");
    return G4_OK;
}

}  // extern "C"
