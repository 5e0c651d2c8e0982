// Types of a served batch's rows (rownorm.hip, linear8.hip, lora.hip) and the
// checks that their entry points share.
#pragma once

#include <initializer_list>

#include "common.h"
#include "row_ranges.h"

namespace g4 {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef int32_t i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr uint32_t kMaxRows = 1u << 22;  // tokens of a batch's buffers

inline uint32_t type_bytes(uint32_t type) { return type == G4_F32 ? 4 : type == G4_E4M3 ? 1 : 2; }
inline bool aligned(const void* p, uint64_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// An operand by its name, for the checks below.
struct Operand {
    const char* name;
    RowRange at;
};
inline Operand rows_operand(const char* name, const void* p, uint32_t type, uint64_t n, uint64_t stride, uint64_t rows) {
    return {name, {p, n * type_bytes(type), stride * type_bytes(type), rows}};
}
// What a call writes shares no memory with what other workgroups of it may still read, or write.
inline int apart_check(const char* what, const Operand& written, std::initializer_list<Operand> others) {
    for (const Operand& o : others)
        if (rows_meet(written.at, o.at)) return fail(G4_EINVAL, "%s: %s lies over %s", what, written.name, o.name);
    return G4_OK;
}

__device__ __forceinline__ uint16_t f2bf(float x) { return __builtin_bit_cast(uint16_t, static_cast<__bf16>(x)); }
__device__ __forceinline__ float bf2f(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }

// Two f32 as e4m3, nearest even, in the low half; values past 448 become 448 (the conversion alone makes them NaN).
__device__ __forceinline__ uint32_t e4m3_pair(float x, float y) {
    x = __builtin_amdgcn_fmed3f(x, -448.0f, 448.0f);
    y = __builtin_amdgcn_fmed3f(y, -448.0f, 448.0f);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x, y, 0, false) & 0xFFFFu;
}

// Two f32 in one of the 16-bit types. Each is rounded to f32 where it was computed: fused with the product before it,
// the rounding to f16 would differ from that of other stores of the same value.
__device__ __forceinline__ uint32_t pair16(float x, float y, uint32_t type) {
    asm("" : "+v"(x), "+v"(y));
    const f32x2 v = {x, y};
    return type == G4_F16 ? __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2))
                          : __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}

// Four outputs of a row in the row's type, at any element: one store, or one each of those below `left` at the row's end. The
// chip takes 16 and 8 bytes at any element's address (a store an element where rows are not aligned to it: 1144 tokens by 5039
// f32 outputs of 272 29.8 us against 17.3, 4096 by 12287 f16 ones of 1536 185 against 120).
typedef f32x4 f32x4_any __attribute__((aligned(4)));
typedef u16x4 u16x4_any __attribute__((aligned(2)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));  // eight of 16 bits
__device__ __forceinline__ void store4(void* out, uint32_t type, uint64_t at, f32x4 v, unsigned left) {
    if (type == G4_F32) {
        float* o = static_cast<float*>(out) + at;
        if (left >= 4) *(__attribute__((address_space(1))) f32x4_any*)o = v;
        else
            for (unsigned i = 0; i < 4; i++)
                if (i < left) stg<float>(o + i, v[i]);
        return;
    }
    const uint32_t lo = pair16(v[0], v[1], type), hi = pair16(v[2], v[3], type);
    const u16x4 h = {(uint16_t)lo, (uint16_t)(lo >> 16), (uint16_t)hi, (uint16_t)(hi >> 16)};
    uint16_t* o = static_cast<uint16_t*>(out) + at;
    if (left >= 4) *(__attribute__((address_space(1))) u16x4_any*)o = h;
    else
#pragma unroll
        for (unsigned i = 0; i < 4; i++)
            if (i < left) stg<uint16_t>(o + i, h[i]);
}
__device__ __forceinline__ f32x4 load4(const void* in, uint32_t type, uint64_t at, unsigned left) {
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (type == G4_F32) {
        const float* p = static_cast<const float*>(in) + at;
        if (left >= 4) return *(const __attribute__((address_space(1))) f32x4_any*)p;
#pragma unroll
        for (unsigned i = 0; i < 4; i++)
            if (i < left) v[i] = ldg<float>(p + i);
        return v;
    }
    const uint16_t* p = static_cast<const uint16_t*>(in) + at;
    u16x4 h = {0, 0, 0, 0};
    if (left >= 4) h = *(const __attribute__((address_space(1))) u16x4_any*)p;
    else
#pragma unroll
        for (unsigned i = 0; i < 4; i++)
            if (i < left) h[i] = ldg<uint16_t>(p + i);
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = type == G4_F16 ? h2f(h[i]) : bf2f(h[i]);
    return v;
}


// Where a DMA lane reads that has nothing to read.
static __device__ __attribute__((aligned(16))) const uint32_t kZeros[4] = {0, 0, 0, 0};

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // M0 is a reserved register: clobbering it is what is meant
// 16 bytes a lane from base + its offset, or from its address, to LDS lds + at + 16 lane. No memory clobber: it writes a
// stage that nothing reads before the barrier that waits for it, and reads of other stages may pass it. Wait states that
// the compiler does not put into assembly: one between a scalar write of M0 and the DMA, five between a vector instruction
// that leaves the base in scalar registers and the DMA.
template <unsigned AT>
__device__ __forceinline__ void stage_dma(const void* base, uint32_t off, uint32_t lds) {
    asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds), "n"(AT) : "m0", "scc");
}
template <unsigned AT>
__device__ __forceinline__ void stage_dma(const void* from, uint32_t lds) {
    asm volatile("s_add_u32 m0, %1, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(lds), "n"(AT) : "m0", "scc");
}
// Four bytes a lane to LDS lds + 4 lane.
__device__ __forceinline__ void scale_dma(const void* from, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(from), "s"(lds) : "m0");
}
#pragma clang diagnostic pop

}  // namespace g4
