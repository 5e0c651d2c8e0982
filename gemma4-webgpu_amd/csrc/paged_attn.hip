// Attention of a batch's new tokens (single ones, chains, trees of drafted
// tokens) over a paged cache: g4_paged_attn.
//
// Per query row r = (token, query head of a kv head) and attended cache row i:
//   s_i = scale q.k_i (capped: softcap tanh(s / softcap)), p_i = e^(s_i - m),
//   out = sum p_i v_i / sum p_i, with the running maximum m and sum of an online
//   softmax, f32 throughout; K and V are read once per tile of query rows.
//
// MFMA mapping (v_mfma_f32_16x16x32_f16; lane = 16 g + n), for each 32-row tile of
// the cache, per group of 16 query rows:
//   S^T[16 rows x 16 q] = K[16 x 32 d] Q^T: lane (n, g) supplies 8 elements of K row n,
//     straight from the cache; the query is f16, so products are exact.
//   O^T[16 d x 16 q] += V^T[16 d x 32 rows] P^T: lane (n, g) holds V pieces of rows
//     4g..4g+3 and 16+4g..16+4g+3, the rows whose scores it has, and transposes them in
//     registers. P goes in twice, as its f16 value and the f16 residual, so that an f32 result
//     keeps f32 accuracy (one f16 P alone leaves 2e-4): off by 2^-24 of a weight down to 2^-8 of
//     the largest one, from there on by 2^-32 of that (paged_softmax).
// e4m3 pools are widened to f16 in registers, which is exact.
//
// Two forms. Few query rows a kv head (up to 16, at head_dim 256 up to 32; k_paged_few): the workgroup's
// waves take different cache rows, K and V go from memory to registers, and the cache's bytes bound it. More
// (k_paged_tile): the waves take different query rows of one tile and share K and V rows through LDS, whose
// reads, with the softmax and the transposition, then bound it.
//
// Work split: a (sequence, tile of query rows, kv head) is an item of ceil(rows / 32)
// row tiles; all items' tiles in order are cut into equal shares, one a workgroup,
// whatever the rows, so a ragged batch fills the chip and one long sequence does
// too; few items are cut each by itself (PagedPieces), and short ones not at all
// (paged_whole). Lengths are read on the device (a captured launch serves the next
// step's), every workgroup finds its share by a scan over the items. An item cut
// between workgroups leaves (m, l, o) records that a second launch joins in a fixed
// order. The host knows the longest sequence's new tokens alone, so every sequence
// has that many query tiles in the scan and in the join's grid: one chunk of 1024
// tokens beside 63 single ones (4096 rows each) takes 395 us, as two calls 157.
#include "decode_core.h"
#include "paged.h"

namespace g4 {

constexpr int kPagedWaves = 4;  // of k_paged_few

struct PagedAttnArgs {
    const uint16_t* __restrict__ q;
    float* __restrict__ out;
    const char* __restrict__ k;
    const char* __restrict__ v;
    float* __restrict__ part_o;   // [2 * workgroups][tile rows][HD]
    float* __restrict__ part_ml;  // [2 * workgroups][tile rows][2]
    uint32_t nkh, group;
    uint32_t q_tiles;             // query tiles a sequence and kv head has at most
    int32_t window;               // 0: none
    float qscale;                 // scale * log2(e)
    float cap_scale, cap_log2;    // scale / cap and cap * log2(e); 0: no cap
    uint32_t wgs;                 // workgroups of the attention launch
    uint32_t whole;               // 1: a workgroup an item, nothing is cut
    PagedBatchDev b;
};

// ---- the items ----------------------------------------------------------------

// Row tiles (UR rows) of query tile qt (MQ query rows) of a sequence: [first, first + n), n >= 1
// where it has such a tile, 0 otherwise. hi: one past the last row that any of its
// tokens attends.
struct PagedSpan {
    unsigned first, n, hi;
};
template <int MQ, int UR>
__device__ __forceinline__ PagedSpan paged_span(const PagedAttnArgs& a, const PagedSeq& sq, unsigned qt) {
    PagedSpan s{};
    if (qt * MQ >= sq.n * a.group) return s;
    const unsigned j0 = qt * MQ / a.group;
    const unsigned j1 = min((qt * MQ + MQ - 1) / a.group, sq.n - 1);
    s.hi = min(sq.ctx + (a.b.mask ? sq.n : j1 + 1), paged_rows(a.b));
    unsigned lo = 0;
    if (a.window) {  // a token's position is its row, or given and then at least ctx
        const int at = (int)(sq.ctx + (a.b.positions ? 0u : j0)) - a.window + 1;
        lo = (unsigned)max(at, 0);
    }
    s.first = min(lo, s.hi - 1) / UR;
    s.n = (s.hi + UR - 1) / UR - s.first;
    return s;
}

// Inclusive sum over the wave's lanes: shifts within rows of 16 lanes, then a row's (two rows') last sum
// into the rows behind it.
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned scan_dpp(unsigned x) {  // 0 where no lane is read
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, true);
}
__device__ __forceinline__ unsigned wave_scan(unsigned x) {
    x += scan_dpp<0x111, 0xf>(x);  // row_shr:1
    x += scan_dpp<0x112, 0xf>(x);
    x += scan_dpp<0x114, 0xf>(x);
    x += scan_dpp<0x118, 0xf>(x);
    x += scan_dpp<0x142, 0xa>(x);  // row_bcast:15, rows 1 and 3
    return x + scan_dpp<0x143, 0xc>(x);  // row_bcast:31, rows 2 and 3
}
__device__ __forceinline__ unsigned lane_value(unsigned x, unsigned lane) {
    return __builtin_amdgcn_readlane(x, lane);
}

// x, with whatever is computed from it computed where it stands: lane addresses of a loop's ends would
// otherwise be computed ahead of the loop and held through it.
__device__ __forceinline__ int not_hoisted(int x) {
    asm volatile("" : "+v"(x));
    return x;
}
__device__ __forceinline__ unsigned uniform(unsigned x) { return __builtin_amdgcn_readfirstlane(x); }

// The batch's row tiles, as a wave sees them: lane l holds query tile i0 + l of all
// sequences' (q_tiles each, in order) and its row tiles for all kv heads.
template <int MQ, int UR>
struct PagedScan {
    unsigned total = 0;
    unsigned head = 0, tiles = 0, incl = 0;  // row tiles of one kv head, of all, of the lanes up to this one
    PagedSeq sq{};

    __device__ __forceinline__ static unsigned items(const PagedAttnArgs& a) { return a.b.n_seqs * a.q_tiles; }
    __device__ __forceinline__ void group(const PagedAttnArgs& a, unsigned i0, unsigned lane) {
        const unsigned i = i0 + lane;
        head = 0;
        if (i < items(a)) {
            const bool one = a.q_tiles == 1;
            sq = paged_seq(a.b, one ? i : i / a.q_tiles);
            head = paged_span<MQ, UR>(a, sq, one ? 0u : i % a.q_tiles).n;
        }
        tiles = head * a.nkh;
        incl = wave_scan(tiles);
    }
    __device__ __forceinline__ void run(const PagedAttnArgs& a, unsigned lane) {
        for (unsigned i0 = 0; i0 < items(a); i0 += 64) {
            group(a, i0, lane);
            total += lane_value(incl, 63);
        }
    }
    // Tiles a workgroup takes (the last one fewer).
    __device__ __forceinline__ unsigned share(const PagedAttnArgs& a) const {
        return max((total + a.wgs - 1) / a.wgs, 1u);
    }
};

// Pieces: where every item cut by itself into pieces of about a share still fits the workgroups, no
// workgroup takes the end of one item and the beginning of the next (which costs it the query, the page
// ids, the pipeline's start and a record once more). Lane l: query tile l's. Several query tiles of the same
// cache rows have pieces in a multiple of the XCDs, so that the pieces of the same rows meet in one L2.
// (26 tokens over 8192 rows at head_dim 512: 48 us in shares, 41 in pieces, 56 of 5 tiles an item.)
struct PagedPieces {
    bool fit;
    unsigned n, per, first;  // pieces a kv head, tiles a piece, the first piece's workgroup

    template <int MQ, int UR>
    __device__ __forceinline__ void run(const PagedAttnArgs& a, const PagedScan<MQ, UR>& scan, unsigned share) {
        fit = false;
        if (scan.items(a) > 64) return;  // uniform
        n = (scan.head + share - 1) / share;
        per = share;
        if (a.q_tiles > 1) {
            n = (n + 7) & ~7u;
            per = n ? (scan.head + n - 1) / n : 1u;
        }
        const unsigned incl = wave_scan(n * a.nkh);
        first = incl - n * a.nkh;
        fit = lane_value(incl, 63) <= a.wgs;
    }
};

// An item and where a tile number lies in it.
struct PagedPlace {
    unsigned i;    // sequence * q_tiles + query tile
    unsigned kvh;
    unsigned off;  // tiles of the item before it
    PagedSeq sq;
};
template <int MQ, int UR>
__device__ __forceinline__ PagedPlace paged_place(const PagedAttnArgs& a, PagedScan<MQ, UR>& scan, unsigned u, unsigned lane) {
    PagedPlace p{};
    unsigned before = 0;
    for (unsigned i0 = 0;; i0 += 64) {
        if (scan.items(a) > 64) scan.group(a, i0, lane);
        const unsigned all = lane_value(scan.incl, 63);
        if (u < before + all || i0 + 64 >= scan.items(a)) {
            const unsigned l = __builtin_ctzll(__ballot(scan.incl > u - before) | (1ull << 63));
            const unsigned mine = lane_value(scan.tiles, l), per_head = lane_value(scan.head, l);
            const unsigned rem = u - (before + lane_value(scan.incl, l) - mine);
            p.i = i0 + l;
            p.kvh = rem / per_head;
            p.off = rem % per_head;
            p.sq = PagedSeq{lane_value(scan.sq.start, l), lane_value(scan.sq.n, l), lane_value(scan.sq.ctx, l)};
            return p;
        }
        before += all;
    }
}
// A workgroup's share [u, end) of the batch's tiles and where it begins; false: none is left for it.
template <int MQ, int UR>
__device__ __forceinline__ bool paged_begin(const PagedAttnArgs& a, unsigned lane, PagedPlace& p, unsigned& u, unsigned& end) {
    if (a.whole) {  // one item, counted from its own first tile
        p.i = blockIdx.x;
        p.kvh = p.off = 0;
        if (a.nkh > 1) {
            p.i = blockIdx.x / a.nkh;
            p.kvh = blockIdx.x % a.nkh;
        }
        p.sq = paged_seq(a.b, a.q_tiles > 1 ? p.i / a.q_tiles : p.i);
        u = 0;
        end = paged_span<MQ, UR>(a, p.sq, a.q_tiles > 1 ? p.i % a.q_tiles : 0u).n;
        return end > 0;
    }
    PagedScan<MQ, UR> scan;
    scan.run(a, lane);
    const unsigned share = scan.share(a);
    PagedPieces pc;
    pc.run(a, scan, share);
    if (pc.fit) {
        const uint64_t there = __ballot(pc.n && pc.first <= blockIdx.x);
        if (!there) return false;
        const unsigned l = 63 - __builtin_clzll(there), mine = lane_value(scan.head, l);
        const unsigned n = lane_value(pc.n, l), per = lane_value(pc.per, l), x = blockIdx.x - lane_value(pc.first, l);
        p.i = l;
        p.kvh = 0;
        p.off = x;
        if (a.nkh > 1) {
            p.kvh = x / n;
            p.off = x % n;
        }
        p.off *= per;
        p.sq = PagedSeq{lane_value(scan.sq.start, l), lane_value(scan.sq.n, l), lane_value(scan.sq.ctx, l)};
        u = 0;
        end = p.off < mine ? min(per, mine - p.off) : 0u;
        return end > 0 && p.kvh < a.nkh;  // past the last piece: none
    }
    const uint64_t first = (uint64_t)blockIdx.x * share;
    if (first >= scan.total) return false;
    u = (unsigned)first;
    end = min(u + share, scan.total);
    p = paged_place<MQ, UR>(a, scan, u, lane);
    return true;
}
// The item after p's: the next kv head, or the next query tile that there is.
template <int MQ, int UR>
__device__ __forceinline__ void paged_next(const PagedAttnArgs& a, PagedPlace& p) {
    p.off = 0;
    if (++p.kvh < a.nkh) return;
    p.kvh = 0;
    const unsigned items = a.b.n_seqs * a.q_tiles;
    do {
        p.i++;
        if (p.i >= items) return;
        p.sq = paged_seq(a.b, p.i / a.q_tiles);
    } while (paged_span<MQ, UR>(a, p.sq, p.i % a.q_tiles).n == 0);
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
    for (int c = 0; c < PagedDims<HD, F8>::KP; c++) kr[c] = ldg_stream<u32x4>(base + (off + c * 64u));
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
            vr[b][t] = ldg_stream<u32x4>((t < 4 ? base0 : base1) + (off + (uint32_t)(t & 3) * row_bytes + b * 256u));
}

// O^T += V^T P^T for piece block b of V, all query groups. Word w of a row's piece holds
// elements (2w, 2w + 1) (f16) or 4w .. 4w + 3 (e4m3): acc tile b E + e takes element e of
// every lane's piece, so its rows are d = 16 E b + E (row) + e.
template <int HD, int C, bool F8>
__device__ __forceinline__ void paged_pv(int b, const u32x4 (&vr)[8], const f16x8 (&hi)[C], const f16x8 (&lo)[C],
                                         f32x4 (&acc)[C][PagedDims<HD, F8>::NO]) {
    using D = PagedDims<HD, F8>;
#pragma unroll
    for (int w = 0; w < 4; w++)
#pragma unroll
        for (int h = 0; h < (F8 ? 2 : 1); h++) {
            uint32_t x[8];
#pragma unroll
            for (int t = 0; t < 8; t++) x[t] = F8 ? fp8x2_f16(vr[t][w], h) : vr[t][w];
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
        }
}

// Words of V pieces whose elements are Inf or NaN (exponent all ones; e4m3: NaN alone): their places, as
// the elements' top bits.
template <bool F8>
__device__ __forceinline__ uint32_t odd_elements(uint32_t w) {
    return F8 ? ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u : ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
}

// Takes Inf and NaN out of a lane's V pieces; returns the rows that had some, as bits 4 t + g
// over the wave's lane groups.
template <bool F8>
__device__ __forceinline__ uint32_t paged_take_odd(u32x4 (&vr)[8]) {
    uint32_t odd = 0;
#pragma unroll
    for (int t = 0; t < 8; t++)
#pragma unroll
        for (int w = 0; w < 4; w++) odd |= odd_elements<F8>(vr[t][w]);
    if (!__any(odd != 0)) return 0;  // uniform
    uint32_t rows = 0;
#pragma unroll
    for (int t = 0; t < 8; t++) {
        uint32_t any = 0;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const uint32_t o = odd_elements<F8>(vr[t][w]);
            any |= o;
            vr[t][w] &= ~((o >> (F8 ? 7 : 15)) * (F8 ? 0xffu : 0xffffu));  // each odd element's bit 0, times all ones
        }
        const uint64_t lanes = __ballot(any != 0);
#pragma unroll
        for (int g = 0; g < 4; g++) rows |= ((lanes >> (16 * g) & 0xffff) ? 1u : 0u) << (4 * t + g);
    }
    return rows;
}

// What one V row's Inf and NaN elements give the outputs of a lane whose column attends the row.
template <int HD, bool F8>
__device__ __forceinline__ void paged_add_odd(const char* row, int g, bool attends, f32x4 (&acc)[PagedDims<HD, F8>::NO]) {
    using D = PagedDims<HD, F8>;
    g = not_hoisted(g);
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

// Waits for the wave's loads (vmcnt 0, the other counters as they are). Stands at the end of code that
// runs now and then and loads: left to the compiler, the wait would be put where that code's paths meet
// the common one, and there wait for every request of the pipeline, tile after tile.
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0F70); }

// ---- a row tile against a lane's query columns ------------------------------------

// Column n of the lane's query groups (group c: 16 query rows from r0 on).
template <int C>
struct PagedCols {
    unsigned j[C];  // new-token index; ~0: no row

    __device__ __forceinline__ void load(const PagedAttnArgs& a, const PagedSeq& sq, unsigned r0) {
#pragma unroll
        for (int c = 0; c < C; c++) j[c] = r0 + 16 * c < sq.n * a.group ? (r0 + 16 * c) / a.group : ~0u;
    }
    // seen[c] bit t: the column attends the lane's row t of the tile at kt0 (rows 4g + t, and
    // 16 + 4g + t - 4 from t = 4 on). dead: the rows nobody may read (past the last, or without a page).
    // A column's committed rows are a range, and its new ones a range or bits of one mask word; masks of
    // more words, and windows that may leave a drafted row behind, are looked up row by row.
    __device__ __forceinline__ void look(const PagedAttnArgs& a, const PagedSeq& sq, unsigned hi, unsigned kt0, int g, bool ok0,
                                         bool ok1, unsigned (&seen)[C], unsigned& dead) const {
        g = not_hoisted(g);
        const int row0 = (int)kt0 + 4 * g, row1 = row0 + 16, ctx = (int)sq.ctx;
        int first[C];  // the first row inside the column's window, for rows that are their own position
        uint64_t word[C];
        bool rows_one_by_one = a.b.mask && a.b.mask_words > 1;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const unsigned jj = j[c] != ~0u ? j[c] : 0u, tok = sq.start + jj;
            const int pos = a.window && a.b.positions ? max(a.b.positions[tok], 0) : ctx + (int)jj;
            first[c] = a.window ? max(pos - a.window + 1, 0) : 0;
            word[c] = a.b.mask ? a.b.mask[(uint64_t)tok * a.b.mask_words] : 0;
            // Drafted rows have positions from ctx on: a window that begins before has them all.
            rows_one_by_one |= __any(a.window && a.b.positions && first[c] > ctx) != 0;
        }
        wait_loads();
        const unsigned live = (ok0 ? rows_below((int)hi - row0) : 0u) | (ok1 ? rows_below((int)hi - row1) : 0u) << 4;
        dead = live ^ 0xffu;
        if (rows_one_by_one) {  // uniform
            one_by_one(a, sq, row0, first, live, seen);
            return;
        }
#pragma unroll
        for (int c = 0; c < C; c++) {
            unsigned s;
            if (a.b.mask) {  // committed rows, then the mask's bits; rows from ctx on are inside the window (below) or
                             // their own positions
                const unsigned in0 = rows_below(ctx - row0), in1 = rows_below(ctx - row1);
                s = in0 | in1 << 4;
                s |= (bits_from(word[c], row0 - ctx) & ~in0) | (bits_from(word[c], row1 - ctx) & ~in1) << 4;
            } else {
                const int end = ctx + (int)j[c] + 1;  // ctx for a column that is none, which the last line clears
                s = rows_below(end - row0) | rows_below(end - row1) << 4;
            }
            if (a.window) {
                // With positions, drafted rows are all inside (above).
                const int from = a.b.positions ? min(first[c], ctx) : first[c];
                s &= ~(rows_below(from - row0) | rows_below(from - row1) << 4);
            }
            seen[c] = j[c] != ~0u ? s & live : 0u;
        }
    }
    // Bits t of 4 rows with t < n.
    __device__ __forceinline__ static unsigned rows_below(int n) { return (1u << min(max(n, 0), 4)) - 1u; }
    // Bits at .. at + 3 of a mask word; those outside it are 0.
    __device__ __forceinline__ static unsigned bits_from(uint64_t word, int at) {
        const uint64_t x = at >= 0 ? word >> min(at, 63) : word << min(-at, 63);
        return at > -4 && at < 64 ? (unsigned)x & 15u : 0u;
    }
    __device__ __forceinline__ void one_by_one(const PagedAttnArgs& a, const PagedSeq& sq, int row0, const int (&first)[C],
                                               unsigned live, unsigned (&seen)[C]) const {
#pragma unroll
        for (int c = 0; c < C; c++) seen[c] = 0;
#pragma unroll 1
        for (int t = 0; t < 8; t++) {
            if (!(live >> t & 1)) continue;
            const unsigned row = (unsigned)row0 + (t < 4 ? t : 12 + t);
            const unsigned dj = row - sq.ctx;  // the new-token index, for rows from ctx on
            int rpos = (int)row;
            if (row >= sq.ctx && a.window && a.b.positions) rpos = max(a.b.positions[sq.start + dj], 0);
#pragma unroll
            for (int c = 0; c < C; c++) {
                bool ok = j[c] != ~0u;
                if (row >= sq.ctx) {
                    if (a.b.mask) {
                        if (ok) ok = (a.b.mask[(uint64_t)(sq.start + j[c]) * a.b.mask_words + (dj >> 6)] >> (dj & 63)) & 1;
                    } else {
                        ok = ok && dj <= j[c];
                    }
                }
                seen[c] |= (ok && (!a.window || rpos >= first[c]) ? 1u : 0u) << t;
            }
        }
        wait_loads();
    }
};

// How a wave takes a 32-row tile: not at all, as it is, or masked.
enum PagedTake { kSkip, kClear, kMasked };

// The online softmax of NX tiles' scores (log2 units), together; P leaves as f16 and its residual, both
// rounded to nearest. P is 2^(score - m_run), and m_run lies kPagedLift below the maximum that it was set at and
// moves once a score is kPagedMove above that: P stays within f16 (2^15 at most), and half of f16's least step,
// 2^-25, is at most 2^-32 of the largest weight. That counts where many rows lie far below the largest, as behind
// an attention sink: 2^17 of them are off by 3e-5 in all at most, and as P is rounded to nearest mostly by far less
// (relative to the maximum itself and truncated, the weights of 16384 rows 17 nats below one lost 6e-4 of the output).
// A larger lift leaves less to the move, and outputs are rescaled more often (64 sequences of 8 tokens, 1024 tokens over
// 7001 rows: 7 and 8 take 0 and 1 % longer than no lift, 11 and 4 2.5 %). The factor is the same in l, o and the records, and falls out of
// their quotient.
constexpr float kPagedLift = 7.0f, kPagedMove = 8.0f;
template <int HD, int C, bool F8, int NX>
__device__ __forceinline__ void paged_softmax(const PagedAttnArgs& a, const f32x4 (&sc)[NX][C][2], const unsigned (&seen)[NX][C],
                                              const PagedTake (&how)[NX], float (&m_run)[C], float (&l_run)[C],
                                              f32x4 (&acc)[C][PagedDims<HD, F8>::NO], f16x8 (&hi)[NX][C], f16x8 (&lo)[NX][C]) {
#pragma unroll
    for (int c = 0; c < C; c++) {
        float sv[NX][8];
        float tmax = -INFINITY;
#pragma unroll
        for (int x = 0; x < NX; x++) {
            if (a.cap_log2 > 0.0f) {  // uniform, once a tile
                float far = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    sv[x][i] = sc[x][c][i >> 2][i & 3] * a.cap_scale;
                    far = fmaxf(far, fabsf(sv[x][i]));
                }
                if (__any(far >= 0.5f)) {  // scores beyond half the cap are few
#pragma unroll
                    for (int i = 0; i < 8; i++) sv[x][i] = a.cap_log2 * tanh_f32(sv[x][i]);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i++) sv[x][i] = a.cap_log2 * tanh_near(sv[x][i]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) sv[x][i] = sc[x][c][i >> 2][i & 3] * a.qscale;
            }
            if (how[x] != kClear) {
                const unsigned keep = how[x] == kSkip ? 0u : seen[x][c];
#pragma unroll
                for (int i = 0; i < 8; i++) sv[x][i] = keep >> i & 1 ? sv[x][i] : -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < 8; i++) tmax = fmaxf(tmax, sv[x][i]);
        }
        tmax = max_xor16(tmax);  // the column's rows lie in four lane groups
        tmax = max_xor32(tmax);
        const bool move = tmax > m_run[c] + (kPagedLift + kPagedMove);
        if (__any(move)) {
            const float m_new = move ? tmax - kPagedLift : m_run[c];
            const float alpha = move ? __builtin_amdgcn_exp2f(m_run[c] - m_new) : 1.0f;
            m_run[c] = m_new;
            l_run[c] *= alpha;
#pragma unroll
            for (int i = 0; i < PagedDims<HD, F8>::NO; i++) acc[c][i] *= alpha;
        }
        const float base = m_run[c] == -INFINITY ? 0.0f : m_run[c];
#pragma unroll
        for (int x = 0; x < NX; x++)
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const float p0 = __builtin_amdgcn_exp2f(sv[x][i] - base), p1 = __builtin_amdgcn_exp2f(sv[x][i + 1] - base);
                l_run[c] += p0 + p1;
                const f16x2 h = __builtin_convertvector((f32x2{p0, p1}), f16x2);
                const f16x2 r = __builtin_convertvector((f32x2{p0 - (float)h[0], p1 - (float)h[1]}), f16x2);
                hi[x][c][i] = h[0];
                hi[x][c][i + 1] = h[1];
                lo[x][c][i] = r[0];
                lo[x][c][i + 1] = r[1];
            }
    }
}

// Page ids of the two 16-row halves of 64 row tiles, lane i the i-th (stride tiles apart from tile0 on).
struct PagedPages {
    unsigned half0, half1;
    __device__ __forceinline__ void load(const PagedAttnArgs& a, const int32_t* table, unsigned tile0, unsigned stride,
                                         unsigned hi, unsigned lane) {
        const unsigned r = (tile0 + stride * lane) * 32;
        half0 = (unsigned)table[min(r, hi - 1) >> a.b.page_shift];
        half1 = (unsigned)table[min(r + 16, hi - 1) >> a.b.page_shift];
    }
};
// Byte offsets of a tile's halves in the pools (page 0 where there is none, ok false).
struct PagedAt {
    uint64_t half0, half1;
    bool ok0, ok1;
};
__device__ __forceinline__ PagedAt paged_at(const PagedAttnArgs& a, const PagedPages& p, unsigned i, unsigned kt0,
                                            uint32_t row_bytes, uint32_t head_off) {
    const unsigned pg0 = lane_value(p.half0, i), pg1 = lane_value(p.half1, i), in = (1u << a.b.page_shift) - 1;
    PagedAt t;
    t.ok0 = pg0 < a.b.num_pages;
    t.ok1 = pg1 < a.b.num_pages;
    t.half0 = (((uint64_t)(t.ok0 ? pg0 : 0u) << a.b.page_shift) + (kt0 & in)) * row_bytes + head_off;
    t.half1 = (((uint64_t)(t.ok1 ? pg1 : 0u) << a.b.page_shift) + ((kt0 + 16) & in)) * row_bytes + head_off;
    return t;
}

__device__ __forceinline__ float paged_inverse(float L) { return L > 0.0f ? 1.0f / L : (L == 0.0f ? 0.0f : L); }

// ---- at most 32 query rows --------------------------------------------------------

// Bound by the cache's bytes: the four waves of a workgroup (512 registers each) take every fourth row tile of its
// share, each with a tile's K and V in registers. The next tile's K is requested when the scores have used this one's,
// its V when the products have. (Eight waves of 256 registers, a tile at a time, for short items that one workgroup has
// whole: 512 sequences of 200 rows f16 31.1 against 29.5 us, e4m3 21.4 against 15.9.)
// Measured: 64 sequences of 1024 to 32768 rows, one token: f16 183 us, 6.3 TB/s; e4m3 104 us, 5.5 TB/s (both read 0.83
// to 0.9 of what a plain read stream does, the rest are ~20 us at the two launches' ends); head_dim 512 f16 364 us,
// 6.3 TB/s, e4m3 194 us, 5.9 TB/s (201 with two tiles ahead); one sequence of 400000 f16 rows 75 us, 5.5 TB/s; five
// tokens of four heads (20 query rows) and a softcap over three sequences of 100001 to 131072 e4m3 rows 75 us, 4.9 TB/s,
// where the work on a tile, 8000 cycles a wave, is the bound: twice the tiles in flight gave nothing (86 us).
template <int HD, int C>
struct PagedFewSmem {
    f16x8 q[C][HD / 32][64];                // score operand, lane-major
    float o[kPagedWaves][HD / 16 * 4][64];  // one query group's outputs, per wave
    float m[kPagedWaves][16 * C], l[kPagedWaves][16 * C];
};

template <int HD, int C, bool F8>
__global__ __launch_bounds__(64 * kPagedWaves, 1) void k_paged_few(const PagedAttnArgs a) {
    using D = PagedDims<HD, F8>;
    constexpr int W = kPagedWaves, MQ = 16 * C, UR = 32;
    static_assert(W == 4, "a wave a row of every four of an output tile");
    __shared__ PagedFewSmem<HD, C> sm;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, g = lane >> 4;
    const unsigned G = a.group;

    PagedPlace at;
    unsigned u, u_end;
    if (!paged_begin<MQ, UR>(a, lane, at, u, u_end)) return;  // uniform
    const uint32_t row_bytes = a.nkh * HD * D::ES;

    bool again = false;
    while (u < u_end) {  // one item or a part of one
        const unsigned i = uniform(at.i);
        const unsigned s = a.q_tiles > 1 ? i / a.q_tiles : i, qt = a.q_tiles > 1 ? i % a.q_tiles : 0u;
        const unsigned kvh = uniform(at.kvh), off = uniform(at.off);
        const PagedSeq sq{uniform(at.sq.start), uniform(at.sq.n), uniform(at.sq.ctx)};
        const PagedSpan sp = paged_span<MQ, UR>(a, sq, qt);
        const unsigned seg = min(sp.n - off, u_end - u);
        const unsigned rows = sq.n * G;
        const uint32_t head_off = kvh * HD * D::ES;
        const int32_t* table = a.b.table + (uint64_t)s * a.b.table_stride;

        // The wave's first tile is requested before the query is read.
        PagedPages pages;
        u32x4 kr[2][D::KP];
        PagedV<HD, F8> vr;
        PagedAt pa{};
        auto load_k = [&](const PagedAt& p) __attribute__((always_inline)) {
            paged_load_k<HD, F8>(a.k + p.half0, row_bytes, n, g, kr[0]);
            paged_load_k<HD, F8>(a.k + p.half1, row_bytes, n, g, kr[1]);
        };
        auto load_v = [&](const PagedAt& p) __attribute__((always_inline)) {
            paged_load_v<HD, F8>(a.v + p.half0, a.v + p.half1, row_bytes, n, g, vr);
        };
        if ((unsigned)wave < seg) {
            pages.load(a, table, sp.first + off + wave, W, sp.hi, lane);
            pa = paged_at(a, pages, 0, (sp.first + off + wave) * 32, row_bytes, head_off);
            load_k(pa);
            load_v(pa);
        }
        if (again) __syncthreads();  // the last segment's combine has read sm
        again = true;
        for (int x = not_hoisted(threadIdx.x); x < C * D::NC * 64; x += 64 * W) {
            const int l = x & 63, ch = (x >> 6) % D::NC, c = (x >> 6) / D::NC;
            const unsigned r = qt * MQ + 16 * c + (l & 15);
            f16x8 v = {};
            if (r < rows)
                v = ldg<f16x8>(a.q + ((uint64_t)(sq.start + r / G) * (a.nkh * G) + kvh * G + r % G) * HD +
                               paged_q_elem<F8>(ch, l >> 4));
            sm.q[c][ch][l] = v;
        }
        PagedCols<C> cols;
        cols.load(a, sq, qt * MQ + (not_hoisted(lane) & 15));
        __syncthreads();

        float m_run[C], l_run[C];
        f32x4 acc[C][D::NO];
#pragma unroll
        for (int c = 0; c < C; c++) {
            m_run[c] = -INFINITY;
            l_run[c] = 0.0f;
#pragma unroll
            for (int x = 0; x < D::NO; x++) acc[c][x] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        // Rows that every column attends: committed, and above every window's start.
        const unsigned clear_lo = !a.window ? 0u : a.b.positions ? sq.ctx : (unsigned)max((int)(sq.ctx + sq.n) - a.window, 0);

        for (unsigned it = 0, t = wave; t < seg; it++, t += W) {
            const unsigned kt0 = (sp.first + off + t) * 32;
            f32x4 sc[1][C][2];
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int h = 0; h < 2; h++) sc[0][c][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ch = 0; ch < D::NC; ch++) {
                const f16x8 k0 = paged_k_chunk<HD, F8>(kr[0], ch), k1 = paged_k_chunk<HD, F8>(kr[1], ch);
#pragma unroll
                for (int c = 0; c < C; c++) {
                    const f16x8 qv = sm.q[c][ch][lane];
                    sc[0][c][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qv, sc[0][c][0], 0, 0, 0);
                    sc[0][c][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qv, sc[0][c][1], 0, 0, 0);
                }
            }
            // The next K into the registers just used (behind a masked tile's work: that needs some).
            const bool more = t + W < seg;
            PagedAt pn{};
            if (more) {
                if (((it + 1) & 63) == 0) pages.load(a, table, sp.first + off + t + W, W, sp.hi, lane);
                pn = paged_at(a, pages, (it + 1) & 63, kt0 + W * 32, row_bytes, head_off);
            }
            const bool clear = kt0 >= clear_lo && kt0 + 32 <= sq.ctx && pa.ok0 && pa.ok1;
            unsigned seen[1][C], dead = 0;
            if (!clear) {
                cols.look(a, sq, sp.hi, kt0, g, pa.ok0, pa.ok1, seen[0], dead);
#pragma unroll
                for (int t8 = 0; t8 < 8; t8++)
                    if (dead >> t8 & 1) {
#pragma unroll
                        for (int b = 0; b < D::VP; b++) vr[b][t8] = u32x4{0u, 0u, 0u, 0u};
                    }
            }
            if (clear && more) load_k(pn);
            f16x8 hi[1][C], lo[1][C];
            const PagedTake how[1] = {clear ? kClear : kMasked};
            paged_softmax<HD, C, F8, 1>(a, sc, seen, how, m_run, l_run, acc, hi, lo);
            // Rows that only some columns attend may hold Inf or NaN, and 0 times those is no 0: they are
            // left out of the products and added to the columns that attend them.
            uint32_t odd_rows = 0;
            if (!clear) {
#pragma unroll
                for (int b = 0; b < D::VP; b++) odd_rows |= paged_take_odd<F8>(vr[b]);
            }
#pragma unroll
            for (int b = 0; b < D::VP; b++) {
                paged_pv<HD, C, F8>(b, vr[b], hi[0], lo[0], acc);
                if constexpr (HD == 512) __builtin_amdgcn_sched_barrier(0);  // block by block: registers
            }
            while (odd_rows) {
                const int bit = __builtin_ctz(odd_rows), t8 = bit >> 2, gg = bit & 3;
                odd_rows &= odd_rows - 1;
#pragma unroll
                for (int c = 0; c < C; c++)
                    paged_add_odd<HD, F8>(a.v + (t8 < 4 ? pa.half0 : pa.half1) + (uint32_t)(4 * gg + (t8 & 3)) * row_bytes, g,
                                          __shfl(seen[0][c], 16 * gg + n) >> t8 & 1, acc[c]);
            }
            if (more) {
                if (!clear) load_k(pn);
                load_v(pn);
            }
            pa = pn;
        }

        const bool whole = seg == sp.n;
        const unsigned slot = 2 * blockIdx.x + (off ? 0u : 1u);  // a part that continues its item, or begins it
        if (seg == 1) {  // one wave had it all (short sequences: one token over 2048 rows 10.7 us, by way of LDS 11.7)
            if (wave == 0) {
                const int el = not_hoisted(lane), en = el & 15, eg = el >> 4;
#pragma unroll
                for (int c = 0; c < C; c++) {
                    float L = add_xor16(l_run[c]);
                    L = add_xor32(L);
                    const unsigned r = qt * MQ + 16 * c + en, rec = 16 * c + en;
                    if (r < rows) {
                        if (whole) {
#pragma unroll
                            for (int x = 0; x < D::NO; x++) acc[c][x] *= paged_inverse(L);
                        }
                        float* dst = whole ? a.out + ((uint64_t)(sq.start + r / G) * (a.nkh * G) + kvh * G + r % G) * HD
                                           : a.part_o + ((uint64_t)slot * MQ + rec) * HD;
                        if (!whole && eg == 0) stg<f32x2>(a.part_ml + ((uint64_t)slot * MQ + rec) * 2, f32x2{m_run[c], L});
#pragma unroll
                        for (int b = 0; b < D::VP; b++)
#pragma unroll
                            for (int j = 0; j < 4; j++)
#pragma unroll
                                for (int e = 0; e < D::E; e += 4) {
                                    const int x = b * D::E + e;
                                    stg<f32x4>(dst + 16 * D::E * b + D::E * (4 * eg + j) + e,
                                               f32x4{acc[c][x][j], acc[c][x + 1][j], acc[c][x + 2][j], acc[c][x + 3][j]});
                                }
                    }
                }
            }
            u += seg;
            if (u < u_end) paged_next<MQ, UR>(a, at);
            continue;
        }
        // The waves' states joined: maxima first, then a query group's outputs at a time.
        const int el = not_hoisted(lane), en = el & 15, eg = el >> 4;
#pragma unroll
        for (int c = 0; c < C; c++) {
            float l = add_xor16(l_run[c]);
            l = add_xor32(l);
            if (eg == 0) {
                sm.m[wave][16 * c + en] = m_run[c];
                sm.l[wave][16 * c + en] = l;
            }
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < C; c++) {
            if (qt * MQ + 16 * c >= rows) break;  // uniform
            float M = -INFINITY, L = 0.0f;
#pragma unroll
            for (int w = 0; w < W; w++) M = fmaxf(M, sm.m[w][16 * c + en]);
            const float base = M == -INFINITY ? 0.0f : M;
#pragma unroll
            for (int w = 0; w < W; w++) L += sm.l[w][16 * c + en] * __builtin_amdgcn_exp2f(sm.m[w][16 * c + en] - base);
            const float f = __builtin_amdgcn_exp2f(m_run[c] - base);
            if (c) __syncthreads();
#pragma unroll
            for (int x = 0; x < D::NO; x++)
#pragma unroll
                for (int j = 0; j < 4; j++) sm.o[wave][x * 4 + j][el] = acc[c][x][j] * f;
            __syncthreads();
            const unsigned r = qt * MQ + 16 * c + en, rec = 16 * c + en;
            if (r < rows) {
                const float inv = whole ? paged_inverse(L) : 1.0f;
                float* dst = whole ? a.out + ((uint64_t)(sq.start + r / G) * (a.nkh * G) + kvh * G + r % G) * HD
                                   : a.part_o + ((uint64_t)slot * MQ + rec) * HD;
                if (!whole && wave == 0 && eg == 0) stg<f32x2>(a.part_ml + ((uint64_t)slot * MQ + rec) * 2, f32x2{M, L});
                const int j = wave;  // of the 4 rows 4g + j of every output tile
#pragma unroll
                for (int b = 0; b < D::VP; b++)
#pragma unroll
                    for (int e = 0; e < D::E; e += 4) {
                        f32x4 x;
#pragma unroll
                        for (int y = 0; y < 4; y++) {
                            const int k = (b * D::E + e + y) * 4 + j;
                            x[y] = ((sm.o[0][k][el] + sm.o[1][k][el]) + (sm.o[2][k][el] + sm.o[3][k][el])) * inv;
                        }
                        stg<f32x4>(dst + 16 * D::E * b + D::E * (4 * eg + j) + e, x);
                    }
            }
        }
        u += seg;
        if (u < u_end) paged_next<MQ, UR>(a, at);
    }
}

// ---- more query rows -----------------------------------------------------------------

// WQ x WK x WD waves: 16 of the tile's 16 WQ query rows each (the query in registers), every WK-th part of a
// row tile of 32 TS rows, with maxima and sums of their own, and a WD-th part of the head: a pair's scores are
// added through LDS, each keeps half of the outputs, so at head_dim 512 two waves fit a SIMD (26 tokens over 8192
// rows 41 -> 37 us). K and V come to LDS by DMA, a row tile's K or its V a slot, NS slots in a ring: K, V, K of
// the next tile and so on, NS - 1 requested ahead; one barrier a slot. A row's 16-byte pieces are stored at
// piece ^ (row % 16), which spreads both operands' reads over all banks (sixteen lanes read sixteen rows of K, or
// sixteen pieces of one row of V). NT: the rows are read by one workgroup alone and bypass the caches (64
// sequences of 8 tokens, pages of 1024, 214 us, without 231).
//
// Measured: 1024 tokens of 8 heads over 7001 rows 139 us, 452 TFLOP/s (0.68 PFLOP/s with the two products of P). A
// tile of 128 query rows and 64 cache rows takes 8600 cycles: 4400 of reading K and V from LDS (128 bytes a
// cycle; each wave reads them whole), of MFMA 3100 beside it, 1150 of softmax, and the rest are the barriers'
// skew and the DMA's issue. 32 query rows a wave would halve the LDS reads, but one wave a SIMD overlaps
// nothing (160 us); scores of the next tile beside this one's softmax (one barrier a tile, half of the waves
// in each order) lost to the lookahead that it takes from the ring (150). 64 sequences of 8 tokens (64 query rows)
// read 5.4 TB/s (209 us).
template <int HD, bool F8, int TS, int NS, int PW>
struct PagedTileSmem {
    unsigned char t[NS][32 * TS][HD * (F8 ? 1 : 2)];
    f32x4 parts[PW][TS][2][64];  // parts of the scores
};

// Waits until at most behind * PER of the wave's DMA requests are outstanding (behind <= MOST, uniform),
// and for the other waves.
template <int MOST, int PER>
__device__ __forceinline__ void dma_barrier(unsigned behind) {
    if constexpr (MOST > 0) {
        if (behind < (unsigned)MOST) {
            dma_barrier<MOST - 1, PER>(behind);
            return;
        }
    }
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(MOST * PER) : "memory");
}

// One LDS-DMA instruction (decode_core.h: lds_dma16_s), for a kernel in which the compiler itself never
// uses M0 (checked in the assembly: its only writes of it are these).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // M0 is a reserved register: clobbering it is what is meant
template <bool NT>
__device__ __forceinline__ void paged_dma(uint32_t voff, const void* sbase, uint32_t lds) {
    if constexpr (NT)
        asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1 nt" ::"v"(voff), "s"(sbase), "s"(lds) : "memory", "m0");
    else
        asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(sbase), "s"(lds) : "memory", "m0");
}
#pragma clang diagnostic pop

template <int HD, int WQ, int WK, int WD, int TS, int NS, bool F8, bool NT>
__global__ __launch_bounds__(64 * WQ * WK * WD, WQ * WK * WD / 4) void k_paged_tile(const PagedAttnArgs a) {
    using D = PagedDims<HD / WD, F8>;  // a wave's part of a row
    constexpr int W = WQ * WK * WD, MQ = 16 * WQ, UR = 32 * TS;
    constexpr int NX = TS / WK;                // 32-row tiles of a slot that a wave works on
    constexpr uint32_t RB = HD * D::ES;        // a row's bytes
    constexpr uint32_t PB = RB / WD;           // a wave's part's
    constexpr uint32_t PPR = RB / 16;          // pieces a row
    constexpr uint32_t RPI = 1024 / RB;        // rows a DMA instruction moves
    constexpr int IH = 16 / RPI;               // instructions 16 rows take
    constexpr int PER = 2 * TS * IH / W;       // of a slot's instructions, a wave's
    static_assert(2 * TS * IH % W == 0 && IH % PER == 0 && TS % WK == 0, "whole instructions, of one half, a wave");
    static_assert((NS - 2) * PER < 64, "outstanding requests are counted in six bits");
    static_assert(WK == 1 || WD == 1, "one of them");
    static_assert(WK == 1 || WQ * HD * 16 * 4 + 2 * MQ * 4 <= NS * UR * (int)RB, "the waves' states are joined in the ring");
    __shared__ __align__(1024) PagedTileSmem<HD, F8, TS, NS, WD == 1 ? 0 : W> sm;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wq = wave % WQ, wk = WK > 1 ? wave / WQ : 0, wd = WD > 1 ? wave / WQ : 0;
    const int n = lane & 15, g = lane >> 4;
    const unsigned G = a.group;

    PagedPlace at;
    unsigned u, u_end;
    if (!paged_begin<MQ, UR>(a, lane, at, u, u_end)) return;  // uniform
    const uint32_t row_bytes = a.nkh * RB;

    // The lane's places in 32 rows: K row n (+ 16), pieces 4 c + g; V rows 4 g + t (+ 16), pieces n (+ 16).
    uint32_t k_at[4], v_at[4];
#pragma unroll
    for (int x = 0; x < 4; x++) {
        k_at[x] = n * RB + (((4 * x + g) ^ n) << 4);
        v_at[x] = (4 * g + x) * RB + ((n ^ (4 * g + x)) << 4);
    }
    // The wave's DMA instructions: its half of a slot, and the lane's bytes in it.
    const unsigned dma_half = wave * PER / IH, inst0 = wave * PER % IH;
    uint32_t dma_off[PER];
#pragma unroll
    for (int x = 0; x < PER; x++) {
        const unsigned r = (inst0 + x) * RPI + lane / PPR;  // of the half's 16 rows
        dma_off[x] = r * row_bytes + ((lane % PPR ^ r) << 4);
    }

    while (u < u_end) {  // one item or a part of one
        const unsigned i = uniform(at.i);
        const unsigned s = a.q_tiles > 1 ? i / a.q_tiles : i, qt = a.q_tiles > 1 ? i % a.q_tiles : 0u;
        const unsigned kvh = uniform(at.kvh), off = uniform(at.off);
        const PagedSeq sq{uniform(at.sq.start), uniform(at.sq.n), uniform(at.sq.ctx)};
        const PagedSpan sp = paged_span<MQ, UR>(a, sq, qt);
        const unsigned seg = min(sp.n - off, u_end - u);
        const unsigned rows = sq.n * G;
        const unsigned w0 = qt * MQ + wq * 16;  // the wave's first query row
        const uint32_t head_off = kvh * RB;
        const int32_t* table = a.b.table + (uint64_t)s * a.b.table_stride;
        // Rows past the wave's own last token are not its business; rows every one of its columns attends
        // need no mask.
        const bool work = w0 < rows;
        const unsigned j0 = w0 / G, j1 = min((w0 + 15) / G, sq.n - 1);
        const unsigned wave_hi = !work ? 0u : a.b.mask ? sp.hi : min(sq.ctx + j1 + 1, sp.hi);
        const unsigned clear_lo = !a.window ? 0u : a.b.positions ? ~0u : (unsigned)max((int)(sq.ctx + j1 + 1) - a.window, 0);
        // sp.hi: a chain may run past the block table, whose last page then ends in the middle of a row tile.
        const unsigned clear_hi = a.b.mask ? sq.ctx : min(sq.ctx + min(j0 + 1, sq.n), sp.hi);

        // The query first: its wait, before the page ids', would otherwise be one for the requests below too.
        f16x8 qr[D::NC];
        {
            const unsigned r = w0 + (not_hoisted(lane) & 15);
            const bool live = r < rows;
            const uint16_t* src = a.q + ((uint64_t)(sq.start + (live ? r / G : 0u)) * (a.nkh * G) + kvh * G + (live ? r % G : 0u)) * HD;
#pragma unroll
            for (int ch = 0; ch < D::NC; ch++) {
                qr[ch] = ldg<f16x8>(src + wd * (HD / WD) + paged_q_elem<F8>(ch, g));
                if (!live) qr[ch] = f16x8{};
            }
        }
        // Page ids: lane l has those of row tile l of 64, for each 16-row half of it; the even and the odd
        // groups of 64.
        unsigned even[2 * TS], odd[2 * TS];
        auto load_pages = [&](unsigned t, unsigned (&p)[2 * TS]) __attribute__((always_inline)) {
            const unsigned r = (sp.first + off + t + (unsigned)lane) * UR;
#pragma unroll
            for (int h = 0; h < 2 * TS; h++) p[h] = (unsigned)table[min(r + 16 * h, sp.hi - 1) >> a.b.page_shift];
            wait_loads();
        };
        load_pages(0, even);
#pragma unroll
        for (int h = 0; h < 2 * TS; h++) odd[h] = 0;
        auto page_of = [&](unsigned t, int h) __attribute__((always_inline)) -> unsigned {  // h: a constant
            const unsigned m = t & 64 ? ~0u : 0u;
            return lane_value((odd[h] & m) | (even[h] & ~m), t & 63);
        };
        // Byte offset in a pool of the half's first row (page 0 where there is none).
        auto half_at = [&](unsigned t, unsigned h, unsigned page) __attribute__((always_inline)) -> uint64_t {
            const unsigned r = (sp.first + off + t) * UR + 16 * h;
            return (((uint64_t)(page < a.b.num_pages ? page : 0u) << a.b.page_shift) + (r & ((1u << a.b.page_shift) - 1))) *
                       row_bytes + head_off;
        };
        // Requests slot j (K of row tile j / 2, or its V) into its place of the ring.
        unsigned ring_in = 0, ring_out = 0;
        auto request = [&](unsigned j) __attribute__((always_inline)) {
            const unsigned t = j >> 1;
            unsigned page = page_of(t, 0);
#pragma unroll
            for (int h = 1; h < 2 * TS; h++) {
                const unsigned p = page_of(t, h);
                page = dma_half == (unsigned)h ? p : page;
            }
            const char* src = uniform_ptr((j & 1 ? a.v : a.k) + half_at(t, dma_half, page));
            const uint32_t dst = (uint32_t)(uintptr_t)&sm.t[ring_in][0][0] + dma_half * 16 * RB + inst0 * 1024;
#pragma unroll
            for (int x = 0; x < PER; x++) paged_dma<NT>(dma_off[x], src, uniform(dst + x * 1024));
            ring_in = ring_in + 1 == NS ? 0 : ring_in + 1;
        };
        // Waits for slot j; every wave has left the one before it then, whose place slot j + NS - 1 takes.
        const unsigned slots = 2 * seg;
        auto take = [&](unsigned j) __attribute__((always_inline)) -> const unsigned char* {
            dma_barrier<NS - 2, PER>(min(slots - 1 - j, (unsigned)(NS - 2)));
            const unsigned ahead = j + NS - 1;
            if (ahead < slots) {
                if ((ahead & 127) == 0) {  // the next 64 tiles' pages; the group before last is done with
                    if (ahead & 128) load_pages(ahead >> 1, odd);
                    else load_pages(ahead >> 1, even);
                }
                request(ahead);
            }
            const unsigned char* p = &sm.t[ring_out][0][0];
            ring_out = ring_out + 1 == NS ? 0 : ring_out + 1;
            return p;
        };
        __syncthreads();  // the last segment's ring is free
#pragma unroll
        for (int j = 0; j < NS - 1; j++)
            if ((unsigned)j < slots) request(j);

        PagedCols<1> cols;
        cols.load(a, sq, w0 + n);
        float m_run[1] = {-INFINITY}, l_run[1] = {0.0f};
        f32x4 acc[1][D::NO];
#pragma unroll
        for (int x = 0; x < D::NO; x++) acc[0][x] = f32x4{0.f, 0.f, 0.f, 0.f};

        for (unsigned t = 0; t < seg; t++) {
            f16x8 hi[NX][1], lo[NX][1];
            f32x4 sc[NX][1][2];
            unsigned seen[NX][1], dead[NX];
            PagedTake how[NX];
            bool some = false;
            const unsigned char* kt = take(2 * t) + wk * NX * 32 * RB + wd * PB;
#pragma unroll
            for (int x = 0; x < NX; x++) {
                const unsigned kt0 = (sp.first + off + t) * UR + (wk * NX + x) * 32;
                how[x] = kSkip;  // uniform
                sc[x][0][0] = sc[x][0][1] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (kt0 >= wave_hi) continue;  // nothing in it for this wave's rows
                some = true;
#pragma unroll
                for (int p = 0; p < D::KP; p++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const u32x4 kv = *reinterpret_cast<const u32x4*>(kt + k_at[p & 3] + (p >> 2) * 256 + (2 * x + h) * 16 * RB);
                        if constexpr (F8) {
#pragma unroll
                            for (int y = 0; y < 2; y++)
                                sc[x][0][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                    __builtin_bit_cast(f16x8, u32x4{fp8x2_f16(kv[2 * y], false), fp8x2_f16(kv[2 * y], true),
                                                                    fp8x2_f16(kv[2 * y + 1], false), fp8x2_f16(kv[2 * y + 1], true)}),
                                    qr[2 * p + y], sc[x][0][h], 0, 0, 0);
                        } else {
                            sc[x][0][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, kv), qr[p], sc[x][0][h], 0, 0, 0);
                        }
                    }
                bool ok0 = true, ok1 = true;
#pragma unroll
                for (int h = 0; h < 2 * TS; h += 2)
                    if (h == 2 * (int)(wk * NX + x)) {
                        ok0 = page_of(t, h) < a.b.num_pages;
                        ok1 = page_of(t, h + 1) < a.b.num_pages;
                    }
                how[x] = kt0 >= clear_lo && kt0 + 32 <= clear_hi && ok0 && ok1 ? kClear : kMasked;
                if (how[x] == kMasked) cols.look(a, sq, sp.hi, kt0, g, ok0, ok1, seen[x], dead[x]);
            }
            if constexpr (WD > 1) {  // the parts' scores, added behind the barrier of V's slot
#pragma unroll
                for (int x = 0; x < NX; x++) {
                    sm.parts[wave][x][0][lane] = sc[x][0][0];
                    sm.parts[wave][x][1][lane] = sc[x][0][1];
                }
            }
            if constexpr (WD == 1)
                if (some) paged_softmax<HD, 1, F8, NX>(a, sc, seen, how, m_run, l_run, acc, hi, lo);
            const unsigned char* vt = take(2 * t + 1) + wk * NX * 32 * RB + wd * PB;
            if constexpr (WD > 1) {
#pragma unroll
                for (int x = 0; x < NX; x++) {
                    sc[x][0][0] += sm.parts[wave ^ WQ][x][0][lane];
                    sc[x][0][1] += sm.parts[wave ^ WQ][x][1][lane];
                }
                if (some) paged_softmax<HD / WD, 1, F8, NX>(a, sc, seen, how, m_run, l_run, acc, hi, lo);
            }
#pragma unroll
            for (int x = 0; x < NX; x++) {
                const unsigned part = wk * NX + x;
                if (how[x] == kSkip) continue;
                uint32_t odd_rows = 0;  // as in k_paged_few
#pragma unroll
                for (int b = 0; b < D::VP; b++) {
                    u32x4 vr[8];
#pragma unroll
                    for (int y = 0; y < 8; y++)
                        vr[y] = *reinterpret_cast<const u32x4*>(vt + v_at[y & 3] + (2 * x + (y >> 2)) * 16 * RB + b * 256);
                    if (how[x] == kMasked) {
#pragma unroll
                        for (int y = 0; y < 8; y++)
                            if (dead[x] >> y & 1) vr[y] = u32x4{0u, 0u, 0u, 0u};
                        odd_rows |= paged_take_odd<F8>(vr);
                    }
                    paged_pv<HD / WD, 1, F8>(b, vr, hi[x], lo[x], acc);
                }
                while (odd_rows) {
                    const int bit = __builtin_ctz(odd_rows), t8 = bit >> 2, gg = bit & 3;
                    odd_rows &= odd_rows - 1;
                    const unsigned half = 2 * part + (t8 >> 2);
                    unsigned page = page_of(t, 0);
#pragma unroll
                    for (int h = 1; h < 2 * TS; h++) {
                        const unsigned p = page_of(t, h);
                        page = half == (unsigned)h ? p : page;
                    }
                    paged_add_odd<HD / WD, F8>(a.v + half_at(t, half, page) + (uint32_t)(4 * gg + (t8 & 3)) * row_bytes + wd * PB, g,
                                          __shfl(seen[x][0], 16 * gg + n) >> t8 & 1, acc[0]);
                }
            }
        }

        const bool whole = seg == sp.n;
        const unsigned slot = 2 * blockIdx.x + (off ? 0u : 1u);  // a part that continues its item, or begins it
        float L = add_xor16(l_run[0]);
        L = add_xor32(L);
        float M = m_run[0];
        if constexpr (WK > 1) {  // the waves of the same query rows joined, in the ring's place
            static_assert(WK == 2, "two parts");
            float* so = reinterpret_cast<float*>(&sm.t[0][0][0]);
            float* sml = so + WQ * HD * 16;
            __syncthreads();
            if (wk == 1) {
#pragma unroll
                for (int x = 0; x < D::NO; x++)
                    *reinterpret_cast<f32x4*>(so + ((wq * D::NO + x) * 64 + lane) * 4) = acc[0][x];
                if (g == 0) {
                    sml[2 * (wq * 16 + n)] = M;
                    sml[2 * (wq * 16 + n) + 1] = L;
                }
            }
            __syncthreads();
            if (wk == 0) {
                const float m2 = sml[2 * (wq * 16 + n)], l2 = sml[2 * (wq * 16 + n) + 1];
                const float m1 = M;
                M = fmaxf(m1, m2);
                const float base = M == -INFINITY ? 0.0f : M;
                const float f1 = __builtin_amdgcn_exp2f(m1 - base), f2 = __builtin_amdgcn_exp2f(m2 - base);
                L = L * f1 + l2 * f2;
#pragma unroll
                for (int x = 0; x < D::NO; x++)
                    acc[0][x] = acc[0][x] * f1 + *reinterpret_cast<const f32x4*>(so + ((wq * D::NO + x) * 64 + lane) * 4) * f2;
            }
        }
        const unsigned r = w0 + (not_hoisted(lane) & 15);
        if (wk == 0 && r < rows) {
            const unsigned rec = r - qt * MQ;
            const float inv = whole ? paged_inverse(L) : 1.0f;
            float* dst = whole ? a.out + ((uint64_t)(sq.start + r / G) * (a.nkh * G) + kvh * G + r % G) * HD
                               : a.part_o + ((uint64_t)slot * MQ + rec) * HD;
            if (!whole && g == 0 && wd == 0) stg<f32x2>(a.part_ml + ((uint64_t)slot * MQ + rec) * 2, f32x2{M, L});
#pragma unroll
            for (int b = 0; b < D::VP; b++)
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int e = 0; e < D::E; e += 4) {
                        const int x = b * D::E + e;
                        stg<f32x4>(dst + wd * (HD / WD) + 16 * D::E * b + D::E * (4 * g + j) + e,
                                   f32x4{acc[0][x][j], acc[0][x + 1][j], acc[0][x + 2][j], acc[0][x + 3][j]} * inv);
                    }
        }
        u += seg;
        if (u < u_end) paged_next<MQ, UR>(a, at);
    }
}

// ---- the join ------------------------------------------------------------------------

// The records of an item that was cut, in P groups of consecutive ones, added in order: the records of
// a group in turn, then the groups. A workgroup takes COLS columns (COLS / 4 threads a group) of
// R = 256 / (P COLS / 4) query rows. Items that are none and items that one workgroup had leave at once.
// Bound by the records' bytes (22 MB of 26 tokens over 8192 rows at head_dim 512: 8 us), or for few of them
// by a launch's start and two dependent reads (4 us).
template <int HD, int MQ, int UR, int P, int COLS>
__global__ __launch_bounds__(256) void k_paged_join(const PagedAttnArgs a) {
    constexpr unsigned TPG = COLS / 4, R = 256 / (P * TPG);
    __shared__ f32x4 so[P > 1 ? 256 : 1];
    __shared__ f32x2 sml[P > 1 ? 256 : 1];
    const unsigned lane = threadIdx.x & 63;
    const unsigned i = blockIdx.x / a.nkh, kvh = blockIdx.x % a.nkh;
    const unsigned s = i / a.q_tiles, qt = i % a.q_tiles;
    const PagedSeq sq = paged_seq(a.b, s);
    const unsigned mine = paged_span<MQ, UR>(a, sq, qt).n;
    if (mine == 0 || qt * MQ + blockIdx.y * R >= sq.n * a.group) return;  // uniform
    PagedScan<MQ, UR> scan;
    unsigned base = 0;  // the item's first tile number
    for (unsigned i0 = 0; i0 < scan.items(a); i0 += 64) {
        scan.group(a, i0, lane);
        if (i >= i0 && i < i0 + 64) base = scan.total + lane_value(scan.incl, i - i0) - lane_value(scan.tiles, i - i0);
        scan.total += lane_value(scan.incl, 63);
    }
    base += kvh * mine;
    const unsigned share = scan.share(a);
    unsigned w0 = base / share, w1 = (base + mine - 1) / share;
    PagedPieces pc;
    pc.run(a, scan, share);
    if (pc.fit) {
        w0 = lane_value(pc.first, i) + kvh * lane_value(pc.n, i);
        w1 = w0 + (mine - 1) / lane_value(pc.per, i);
    }
    if (w0 == w1) return;  // uniform: one workgroup wrote the result
    const unsigned grp = threadIdx.x / TPG % P;
    const unsigned rq = blockIdx.y * R + threadIdx.x / (TPG * P), r = qt * MQ + rq;  // R divides MQ
    const unsigned d = blockIdx.z * COLS + threadIdx.x % TPG * 4;
    // The first record is its workgroup's slot 1, the others continue the item: slot 0.
    auto rec = [&](unsigned w) __attribute__((always_inline)) { return ((uint64_t)2 * w + (w == w0 ? 1u : 0u)) * MQ + rq; };
    const unsigned per = (w1 - w0 + P) / P;  // records a group
    const unsigned first = w0 + grp * per, end = min(first + per, w1 + 1);
    float M = -INFINITY, L = 0.0f;
    f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
    if (r < sq.n * a.group) {  // rows that are none have no records
        constexpr int B = 8;  // records requested at once
        for (unsigned w = first; w < end; w += B) {
            f32x2 ml[B];
            f32x4 x[B];
#pragma unroll
            for (int k = 0; k < B; k++) {
                const uint64_t at = rec(min(w + k, end - 1));
                ml[k] = ldg<f32x2>(a.part_ml + at * 2);
                x[k] = ldg<f32x4>(a.part_o + at * HD + d);
            }
            float m = M;
#pragma unroll
            for (int k = 0; k < B; k++) m = fmaxf(m, ml[k][0]);
            const float ref = m == -INFINITY ? 0.0f : m, f0 = __builtin_amdgcn_exp2f(M - ref);
            L *= f0;
            o *= f0;
#pragma unroll
            for (int k = 0; k < B; k++) {
                const float f = w + k < end ? __builtin_amdgcn_exp2f(ml[k][0] - ref) : 0.0f;
                L += ml[k][1] * f;
                o += x[k] * f;
            }
            M = m;
        }
    }
    if constexpr (P > 1) {
        so[threadIdx.x] = o;
        sml[threadIdx.x] = f32x2{M, L};
        __syncthreads();
        if (grp) return;
        for (unsigned k = 1; k < P; k++) M = fmaxf(M, sml[threadIdx.x + k * TPG][0]);
        const float ref = M == -INFINITY ? 0.0f : M;
        L = 0.0f;
        o = f32x4{0.f, 0.f, 0.f, 0.f};
        for (unsigned k = 0; k < P; k++) {
            const f32x2 ml = sml[threadIdx.x + k * TPG];
            const float f = __builtin_amdgcn_exp2f(ml[0] - ref);
            L += ml[1] * f;
            o += so[threadIdx.x + k * TPG] * f;
        }
    }
    if (r < sq.n * a.group)
        stg<f32x4>(a.out + ((uint64_t)(sq.start + r / a.group) * (a.nkh * a.group) + kvh * a.group + r % a.group) * HD + d,
                   o * paged_inverse(L));
}

// ---- host --------------------------------------------------------------------------

struct PagedPlan {
    unsigned mq, wgs;
    uint64_t q_tiles;  // of a sequence and kv head, at most
    size_t bytes;
};
// Query rows of a tile: 32 (K and V in registers) against a tile of 64 (through LDS), 64 sequences of 4 tokens, e4m3: 122
// and 170 us (f16 195 and 191); 64 against 128, 64 sequences of 8 tokens: 214 and 242 us; 128 against 64, 1024 tokens over
// 7001 rows: 137 and 175 us. At head_dim 512 the registers hold no more than 16 and 64.
static PagedPlan paged_plan(unsigned head_dim, unsigned num_kv_heads, unsigned num_q_heads, const PagedBatchDev& b) {
    PagedPlan p;
    const uint64_t rows = (uint64_t)b.max_tokens * (num_q_heads / num_kv_heads);
    p.mq = rows <= 16 ? 16 : rows <= 32 && head_dim == 256 ? 32 : rows <= 64 || head_dim == 512 ? 64 : 128;
    p.q_tiles = (rows + p.mq - 1) / p.mq;
    p.wgs = device_cus();
    p.bytes = (size_t)2 * p.wgs * p.mq * (head_dim + 2) * sizeof(float);
    return p;
}

// Whether every item goes to one workgroup: its rows are few for certain (by the window, or the block table's
// size), and there are items for the CUs, or for half of them and half as many rows, or one tile or two a wave, so
// that cutting them and joining the parts in a second launch would cost more. (One token, f16, whole / cut: 512
// sequences of 200 rows 30 / 39 us, 256 of a window of 1024 50 / 55, of 200 to 1500 rows 55 / 57; 128 of a window of 512
// 26 / 28, of 1024 43 / 37 but e4m3 27 / 29, four tokens 47 / 49, eight 51 / 56; of 200 to 1500 rows 49 / 34, e4m3 31 / 28,
// four tokens 38 / 43; one sequence over a window of 512 16 / 11, of 1024 31 / 11.)
static bool paged_whole(uint64_t rows, uint64_t items, unsigned cus) {
    if (items >= cus) return rows <= 2048;
    return rows <= (2 * items >= cus ? 1088 : 256);
}

// How the records are joined: few an item, its thread's rows in turn; many, in 16 groups, or in 4 where an item's
// rows fill the chip already. (64 sequences of 8 tokens, 1 / 16 groups: 212 / 240 us; 26 tokens over 8192 rows at
// head_dim 512, 1 / 4 / 16: 37.1 / 34.6 / 36.8; 8 over 32768 rows 43.1 / 33.0 / 29.3; one over 8192 24.2 / 16.9 / 13.4.)
template <int HD, int MQ, int UR>
static void launch_join(const PagedAttnArgs& a, hipStream_t st) {
    if (a.whole) return;
    const unsigned items = a.b.n_seqs * a.q_tiles * a.nkh;
    if (items * 16 >= a.wgs) {
        G4_LAUNCH((k_paged_join<HD, MQ, UR, 1, HD>), dim3(items, MQ * HD / 4 / 256), dim3(256), 0, st, a);
    } else if (MQ <= 32 || items * 128 <= a.wgs) {
        G4_LAUNCH((k_paged_join<HD, MQ, UR, 16, 64>), dim3(items, MQ, HD / 64), dim3(256), 0, st, a);
    } else {
        if constexpr (MQ > 32) G4_LAUNCH((k_paged_join<HD, MQ, UR, 4, 64>), dim3(items, MQ / 4, HD / 64), dim3(256), 0, st, a);
    }
}

template <int HD, bool F8>
static void launch_paged(const PagedAttnArgs& a, const PagedPlan& p, hipStream_t st) {
    const dim3 grid(a.whole ? a.b.n_seqs * a.q_tiles * a.nkh : p.wgs);
    if (p.mq == 16) {
        G4_LAUNCH((k_paged_few<HD, 1, F8>), grid, dim3(64 * kPagedWaves), 0, st, a);
        launch_join<HD, 16, 32>(a, st);
    } else if constexpr (HD == 512) {
        constexpr int TS = F8 ? 2 : 1;
        if (p.q_tiles == 1)
            G4_LAUNCH((k_paged_tile<512, 4, 1, 2, TS, 4, F8, true>), grid, dim3(512), 0, st, a);
        else
            G4_LAUNCH((k_paged_tile<512, 4, 1, 2, TS, 4, F8, false>), grid, dim3(512), 0, st, a);
        launch_join<HD, 64, 32 * TS>(a, st);
    } else if (p.mq == 32) {
        G4_LAUNCH((k_paged_few<256, 2, F8>), grid, dim3(64 * kPagedWaves), 0, st, a);
        launch_join<HD, 32, 32>(a, st);
    } else if (p.mq == 64) {
        G4_LAUNCH((k_paged_tile<256, 4, 2, 1, 2, F8 ? 10 : 5, F8, true>), grid, dim3(512), 0, st, a);
        launch_join<HD, 64, 64>(a, st);
    } else {
        G4_LAUNCH((k_paged_tile<256, 8, 1, 1, 2, F8 ? 10 : 5, F8, false>), grid, dim3(512), 0, st, a);
        launch_join<HD, 128, 64>(a, st);
    }
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
    a.part_ml = a.part_o + (size_t)2 * plan.wgs * plan.mq * cache->head_dim;
    a.nkh = cache->num_kv_heads;
    a.group = p->num_q_heads / cache->num_kv_heads;
    a.window = p->sliding_window > 0x7fffffffu ? 0 : (int32_t)p->sliding_window;  // no position is further on
    a.q_tiles = (uint32_t)plan.q_tiles;
    a.qscale = p->scale * kLog2e;
    a.cap_scale = p->softcap > 0.0f ? p->scale / p->softcap : 0.0f;
    a.cap_log2 = p->softcap * kLog2e;
    a.wgs = plan.wgs;
    const uint64_t cap = (uint64_t)batch->table_stride * cache->page_size;
    const uint64_t span = a.window ? (uint64_t)a.window + a.b.max_tokens : cap;
    a.whole = paged_whole(span < cap ? span : cap, (uint64_t)a.b.n_seqs * a.q_tiles * a.nkh, device_cus());
    hipStream_t st = as_stream(stream);
    const bool f8 = cache->dtype == G4_KV_E4M3;
    if (cache->head_dim == 512) {
        if (f8) launch_paged<512, true>(a, plan, st);
        else launch_paged<512, false>(a, plan, st);
    } else {
        if (f8) launch_paged<256, true>(a, plan, st);
        else launch_paged<256, false>(a, plan, st);
    }
    G4_CHECK_LAUNCH("pagedAttn");
    return G4_OK;
}

}  // extern "C"
