// attn_device.h -- device helpers shared by the kernel sources (attn_kernels.hip,
// paged_kernels.hip): lane reductions, the pair rotation, and the cache element
// types' rows as they are loaded, widened and written.
#pragma once
#include <hip/hip_runtime.h>

#include "attn_args.h"

namespace {

using namespace tmac;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr float kTau = 8.0f;  // lazy-rescale threshold (log2 units): weights stay <= 2^8
constexpr float kNegInf = -__builtin_inff();
constexpr int kLanesPerSlot = 8;
constexpr int kDimsPerLane = kHeadDim / kLanesPerSlot;  // 8
constexpr int kSlots = 64 / kLanesPerSlot;              // 8 (row, kv) slots per wave step

template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __builtin_bit_cast(
        float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xF, 0xF, false));
}

// Sum over the 8 lanes of a slot; every lane receives the same bits.
__device__ __forceinline__ float slot_sum(float x) {
    x += dpp<0xB1>(x);   // quad_perm [1,0,3,2]
    x += dpp<0x4E>(x);   // quad_perm [2,3,0,1]
    x += dpp<0x141>(x);  // row_half_mirror: lane i <- lane 7-i within each 8-lane half row
    return x;
}

// Max over the 8 lanes of a slot; every lane receives the same value.
__device__ __forceinline__ float slot_max(float x) {
    x = fmaxf(x, dpp<0xB1>(x));
    x = fmaxf(x, dpp<0x4E>(x));
    return fmaxf(x, dpp<0x141>(x));
}

// Sum / max over the lanes lane ^ m, m = FIRST, 2 FIRST, ..., 32, without the
// LDS crossbar: DPP inside 16-lane rows (FIRST = 1: the slot patterns above,
// then lane ^ 8 = row_ror:8), then the gfx950 row swaps for lane ^ 16 and
// lane ^ 32 (each returns both swapped registers; the pair's sum or max is the
// same whichever way round they come).  Every lane ends with the same bits.
template <int FIRST>
__device__ __forceinline__ float xor_sum(float x) {
    static_assert(FIRST == 1 || FIRST == 8 || FIRST == 16 || FIRST == 32, "lane groups of 1, 8, 16 or 32");
    if constexpr (FIRST == 1) x = slot_sum(x);
    if constexpr (FIRST <= 8) x += dpp<0x128>(x);
    if constexpr (FIRST <= 16) {
        const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    }
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
template <int FIRST>
__device__ __forceinline__ float xor_max(float x) {
    static_assert(FIRST == 1 || FIRST == 8 || FIRST == 16 || FIRST == 32, "lane groups of 1, 8, 16 or 32");
    if constexpr (FIRST == 1) x = slot_max(x);
    if constexpr (FIRST <= 8) x = fmaxf(x, dpp<0x128>(x));
    if constexpr (FIRST <= 16) {
        const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    }
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Rotation of one adjacent pair, exactly as tmac_gguf.cpp:999-1001 rounds it:
// each product rounded, then the sum/difference rounded (no fused multiply-add).
__device__ __forceinline__ void rotate_pair(float& x0, float& x1, float c, float s) {
#pragma clang fp contract(off)
    const float a = x0 * c;
    const float b = x1 * s;
    const float e = x0 * s;
    const float f = x1 * c;
    x0 = a - b;
    x1 = e + f;
}

// A lane's 8 dims of one head: x[0..3] = dims 4c..4c+3, x[4..7] = dims 32+4c..32+4c+3.
__device__ __forceinline__ void load8(float (&x)[8], const float* __restrict__ p) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    const float4 b = *reinterpret_cast<const float4*>(p + 32);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}

__device__ __forceinline__ void store8(float* __restrict__ p, const float (&x)[8]) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(p + 32) = make_float4(x[4], x[5], x[6], x[7]);
}

// 16-bit caches (bf16 / fp16, the same [row][kv][64] layout): a lane's 8 dims
// are two 8-byte loads, widened exactly to fp32; stores round to nearest even.
template <typename T>
__device__ __forceinline__ void load8(float (&x)[8], const T* __restrict__ p) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    const t4 a = *reinterpret_cast<const t4*>(p);
    const t4 b = *reinterpret_cast<const t4*>(p + 32);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        x[t] = (float)a[t];
        x[4 + t] = (float)b[t];
    }
}

template <typename T>
__device__ __forceinline__ void store8(T* __restrict__ p, const float (&x)[8]) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    const t4 a = {(T)x[0], (T)x[1], (T)x[2], (T)x[3]};
    const t4 b = {(T)x[4], (T)x[5], (T)x[6], (T)x[7]};
    *reinterpret_cast<t4*>(p) = a;
    *reinterpret_cast<t4*>(p + 32) = b;
}

// The value a cache of element type T holds for x: what a later read returns,
// so a row attended from registers matches the row attended from memory.
__device__ __forceinline__ void round8(float (&)[8], const float*) {}
template <typename T>
__device__ __forceinline__ void round8(float (&x)[8], const T*) {
#pragma unroll
    for (int t = 0; t < 8; ++t) x[t] = (float)(T)x[t];
}

__device__ __forceinline__ float half_bits_to_float(unsigned h) {
    return (float)__builtin_bit_cast(_Float16, (unsigned short)h);
}

// Q8_0 cache (TMAC_KV_Q8_0).  The 64 dims of one (row, kv head) form a
// 68-byte "head row": int8 q[64], then the fp16 scales d0 (dims 0..31) and d1
// (dims 32..63).  Those are the two 34-byte GGML Q8_0 blocks of the 64 dims
// (value = q * d, as dequant_q8_0 reads them, tmac_gguf.cpp:240-250) with the
// scales moved behind the values, so each lane's 4-dim runs are aligned
// 4-byte words.
struct q8_0_t {};

// Byte geometry of one head row of a cache of element type T.
template <typename T>
struct CacheFmt {
    static constexpr int kHeadBytes = kHeadDim * (int)sizeof(T);
    static constexpr int kDimBytes = (int)sizeof(T);
};
template <>
struct CacheFmt<q8_0_t> {
    static constexpr int kHeadBytes = kQ8HeadBytes;
    static constexpr int kDimBytes = 1;
};

// 4-bit pages (TMAC_KV_Q4_PAGES).  A (page, kv head) is one block of kQ4Block
// bytes, 512 of codes and 32 fp16 scales, laid out for the product that reads
// it: lane l of a wave takes the eight code bytes from 8 l on, K as the operand
// (row l % 16, dims 16 (l / 16) ..), V as the operand (dims l % 16 + 16 b, four
// rows from 4 (l / 16) on), with no exchange between lanes.  A byte holds two
// dims of one row, so that rows are written without reading what is there.
//   K  byte 8 (16 g + row) + 4 m + c: dims d = 16 g + 8 m + 4 (c & 1) + (c >> 1) and d + 2
//      scale of (row, dims 32 half ..): half word 256 + 16 half + row
//   V  byte 8 (16 (row / 4) + i) + 4 p + {0, 2, 1, 3}[row % 4]: dims 32 p + i and 32 p + i + 16
//      scale: half word 256 + 8 (row / 4) + 4 half + row % 4
// value = (code - 8) * scale.  A scale has 7 significant bits and is 0 or at
// least 2^-14, so that a value is exact in fp16 (4 + 7 bits), and so is a
// sixteenth of its scale.
struct q4_t {};
constexpr int kQ4Block = 576;

// Byte geometry of pages: from row to row of a head, of a page, and of head h in its page.
template <typename T>
struct PageFmt {
    __device__ static size_t row(int kv) { return (size_t)kv * CacheFmt<T>::kHeadBytes; }
    __device__ static size_t page(int kv) { return kPageRows * row(kv); }
    __device__ static size_t head(int h) { return (size_t)h * CacheFmt<T>::kHeadBytes; }
};
struct q4_pair_t {};  // the same pages, for at most 8 query heads a kv head (Own<q4_pair_t>)
template <>
struct PageFmt<q4_t> {
    __device__ static size_t row(int) { return 0; }
    __device__ static size_t page(int kv) { return (size_t)kv * kQ4Block; }
    __device__ static size_t head(int h) { return (size_t)h * kQ4Block; }
};
template <>
struct PageFmt<q4_pair_t> : PageFmt<q4_t> {};

// This lane's 8 dims of a cache head row as loaded (raw words): fp32 8
// floats, 16-bit 4 words, Q8_0 the two 4-byte runs plus the scale word.
// Prefetch buffers hold raw rows and are widened where they are used, so the
// wait for a load sits at its use, not right behind the load.
template <typename T>
struct RawRow {
    unsigned w[sizeof(T) == 2 ? 4 : 3];
};
template <>
struct RawRow<float> {
    float w[8];
};

// A load of a cache word: non-temporal (the `nt` cache policy) when NT.
template <bool NT, typename V>
__device__ __forceinline__ V ld(const char* p) {
    if constexpr (NT)
        return __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
    else
        return *reinterpret_cast<const V*>(p);
}

// p points at the lane's dim 4c of a head row.  The group kernel reads every
// cache row once per launch, so it streams them non-temporally (NT): at
// config 3 that moved the fp32 decode from 185 to 170 us (72% -> 79% of HBM
// peak), the streamed rows no longer displacing useful lines.  The head
// kernel reads each row once per query head, through L2: temporal loads.
template <typename T, bool NT>
__device__ __forceinline__ void load_raw(RawRow<T>& r, const char* p, int c) {
    typedef float f32x4_t __attribute__((ext_vector_type(4)));
    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
    if constexpr (sizeof(T) == 4) {
        const f32x4_t a = ld<NT, f32x4_t>(p);
        const f32x4_t b = ld<NT, f32x4_t>(p + 32 * sizeof(float));
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            r.w[t] = a[t];
            r.w[4 + t] = b[t];
        }
    } else if constexpr (sizeof(T) == 2) {
        const u32x2 a = ld<NT, u32x2>(p);
        const u32x2 b = ld<NT, u32x2>(p + 32 * sizeof(T));
        r.w[0] = a[0];
        r.w[1] = a[1];
        r.w[2] = b[0];
        r.w[3] = b[1];
    } else {
        r.w[0] = ld<NT, unsigned>(p);               // dims 4c..4c+3
        r.w[1] = ld<NT, unsigned>(p + 32);          // dims 32+4c..32+4c+3
        r.w[2] = ld<NT, unsigned>(p + 64 - 4 * c);  // d0 | d1 << 16
    }
}

// Raw row -> fp32, exactly.
template <typename T>
__device__ __forceinline__ void widen(float (&x)[8], const RawRow<T>& r) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int t = 0; t < 8; ++t) x[t] = r.w[t];
    } else if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            if constexpr (__is_same(T, __bf16)) {
                x[2 * t] = __builtin_bit_cast(float, r.w[t] << 16);
                x[2 * t + 1] = __builtin_bit_cast(float, r.w[t] & 0xFFFF0000u);
            } else {
                x[2 * t] = half_bits_to_float(r.w[t] & 0xFFFFu);
                x[2 * t + 1] = half_bits_to_float(r.w[t] >> 16);
            }
        }
    } else {
        const float d0 = half_bits_to_float(r.w[2] & 0xFFFFu), d1 = half_bits_to_float(r.w[2] >> 16);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            x[t] = (float)(signed char)(r.w[0] >> (8 * t)) * d0;  // |q| <= 127, 11-bit d: exact product
            x[4 + t] = (float)(signed char)(r.w[1] >> (8 * t)) * d1;
        }
    }
}

template <typename T, bool NT>
__device__ __forceinline__ void load_row(float (&x)[8], const char* p, int c) {
    RawRow<T> r;
    load_raw<T, NT>(r, p, c);
    widen<T>(x, r);
}

// fp16 bits of a Q8_0 scale exactly as the reference's converter writes them
// (scripts/extract_tmac.py:53-74): exponent rebased, mantissa truncated to 10
// bits, magnitudes below fp16's normal range flushed to 0, exponents above
// its range turned into infinity.
__device__ __forceinline__ unsigned f16_bits_trunc(float v) {
    const unsigned u = __builtin_bit_cast(unsigned, v);
    const unsigned e = (u >> 23) & 0xFFu;
    if ((u & 0x7FFFFFFFu) == 0 || e == 0) return 0;
    const unsigned s = (u >> 31) << 15;
    if (e >= 0x8Fu) return s | (31u << 10);
    if (e <= 0x70u) return s;
    return s | ((e - 112u) << 10) | ((u & 0x7FFFFFu) >> 13);
}

// One lane's 4 dims of a 32-dim block quantized as quantize_q8_0_block does
// (scripts/extract_tmac.py:159-173): d = amax / 127 (1 when amax < 1e-10),
// q = x / d rounded half to even, the scale stored as f16_bits_trunc(d).
// amax is the block's max |x|.  Returns the 4 bytes; x becomes what the cache
// then holds, q * fp16(d).
__device__ __forceinline__ unsigned quant4(float* x, float amax, unsigned& dbits) {
    const float d = amax < 1e-10f ? 1.0f : amax / 127.0f;  // IEEE division (hipcc default)
    dbits = f16_bits_trunc(d);
    const float dq = half_bits_to_float(dbits);
    unsigned packed = 0;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int qv = (int)__builtin_rintf(x[t] / d);
        packed |= ((unsigned)qv & 0xFFu) << (8 * t);
        x[t] = (float)qv * dq;
    }
    return packed;
}

// Rounds x (this lane's 8 dims of a new cache head row) to the value a cache
// of type T holds and, if `store`, writes it at p (the lane's dim 4c).
template <typename T>
__device__ __forceinline__ void put_row(float (&x)[8], char* p, int, bool store) {
    round8(x, static_cast<const T*>(nullptr));
    if (store) store8(reinterpret_cast<T*>(p), x);
}
// Q8_0: the 8 lanes of a slot hold the head row's 64 dims and must all call
// (the block maxima are reduced across them); lane 0 writes the scales.
template <>
__device__ __forceinline__ void put_row<q8_0_t>(float (&x)[8], char* p, int c, bool store) {
    float a0 = 0.f, a1 = 0.f;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        a0 = fmaxf(a0, fabsf(x[t]));
        a1 = fmaxf(a1, fabsf(x[4 + t]));
    }
    a0 = slot_max(a0);
    a1 = slot_max(a1);
    unsigned d0, d1;
    const unsigned lo = quant4(x, a0, d0);
    const unsigned hi = quant4(x + 4, a1, d1);
    if (store) {
        *reinterpret_cast<unsigned*>(p) = lo;
        *reinterpret_cast<unsigned*>(p + 32) = hi;
        if (c == 0) *reinterpret_cast<unsigned*>(p + 64) = d0 | (d1 << 16);
    }
}

// RoPE on a lane's 8 dims.  Pairs (d, d+1), d even, never straddle a lane:
// dims 4c..4c+3 are pairs 2c, 2c+1 and dims 32+4c.. are pairs 16+2c, 17+2c.
__device__ __forceinline__ void rope8(float (&x)[8], const float2* __restrict__ cs_row, int c) {
    const float4 t0 = *reinterpret_cast<const float4*>(cs_row + 2 * c);
    const float4 t1 = *reinterpret_cast<const float4*>(cs_row + 16 + 2 * c);
    rotate_pair(x[0], x[1], t0.x, t0.y);
    rotate_pair(x[2], x[3], t0.z, t0.w);
    rotate_pair(x[4], x[5], t1.x, t1.y);
    rotate_pair(x[6], x[7], t1.z, t1.w);
}

__device__ __forceinline__ unsigned bf16_pair(float a, float b) {
    const bf16x2 v = {(__bf16)a, (__bf16)b};  // round to nearest even
    return __builtin_bit_cast(unsigned, v);
}

// Max / sum over the four lanes l % 16 + 16 * k (k = 0..3) of a wave, via the
// gfx950 row and half-wave swaps (each returns both swapped registers; the
// reduction of the pair is the same whichever way round they come).
__device__ __forceinline__ float max4_rows(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum4_rows(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

typedef __attribute__((address_space(4))) const int32_t* const_i32_ptr;

typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((__vector_size__(4 * sizeof(__bf16)))) __bf16 bf16x4_v;
typedef __attribute__((address_space(3))) bf16x4_v* lds_bf16x4_ptr;
typedef __attribute__((__vector_size__(4 * sizeof(__fp16)))) __fp16 f16x4_v;
typedef __attribute__((address_space(3))) f16x4_v* lds_f16x4_ptr;

// The 16-bit element types of the MFMA decode: operand types, the matching
// MFMAs and transposed LDS read, and packing of fp32 pairs (nearest even).
//   bf16: fp32's exponent range, so q and P are split as they are.
//   fp16: q is scaled per column by a power of two (its largest |value| to
//   [2^14, 2^15)) and P by 2^7 before splitting, so the split parts stay in
//   fp16's normal range; both scales are undone exactly after the MFMAs.
template <typename T>
struct MMath;
template <>
struct MMath<__bf16> {
    typedef bf16x8 v8;
    typedef i16x4 v4;
    static constexpr bool kScaleQ = false;
    static constexpr int kQParts = 3;  // 16-bit parts of an fp32 query element
    static constexpr float kPScale = 1.0f;
    __device__ static unsigned pack2(float a, float b) { return bf16_pair(a, b); }
    __device__ static float lo(unsigned w) { return __uint_as_float(w << 16); }
    __device__ static float hi(unsigned w) { return __uint_as_float(w & 0xffff0000u); }
    __device__ static f32x4 mfma32(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    __device__ static v8 cat(v4 a, v4 b) { return __builtin_bit_cast(v8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7)); }
    __device__ static v4 read_tr(char* p) {
        return __builtin_bit_cast(v4, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4_ptr)p));
    }
};
template <>
struct MMath<_Float16> {
    typedef f16x8 v8;
    typedef f16x4 v4;
    static constexpr bool kScaleQ = true;
    static constexpr int kQParts = 2;
    static constexpr float kPScale = 128.0f;
    __device__ static unsigned pack2(float a, float b) {
        const f16x2 v = {(_Float16)a, (_Float16)b};
        return __builtin_bit_cast(unsigned, v);
    }
    __device__ static float lo(unsigned w) { return half_bits_to_float(w & 0xffffu); }
    __device__ static float hi(unsigned w) { return half_bits_to_float(w >> 16); }
    __device__ static f32x4 mfma32(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    __device__ static v8 cat(v4 a, v4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }
    __device__ static v4 read_tr(char* p) {
        return __builtin_bit_cast(v4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_f16x4_ptr)p));
    }
};

// Four int8 (one word) -> four bf16 (two words, element 2i in the low half), exactly.
__device__ __forceinline__ u32x2 i8x4_to_bf16(unsigned w) {
    const float f0 = (float)(signed char)w, f1 = (float)(signed char)(w >> 8);
    const float f2 = (float)(signed char)(w >> 16), f3 = (float)(signed char)(w >> 24);
    return u32x2{__builtin_amdgcn_perm(__float_as_uint(f1), __float_as_uint(f0), 0x07060302u),
                 __builtin_amdgcn_perm(__float_as_uint(f3), __float_as_uint(f2), 0x07060302u)};
}

// Four int8 (one word) -> four fp16 (two words, element 2i in the low half),
// exactly: byte b becomes u = b ^ 0x80 = b + 128, the fp16 with bits
// 0x6400 | u is 1024 + u, and subtracting 1152 (packed) leaves b.
__device__ __forceinline__ u32x2 i8x4_to_f16(unsigned w) {
    const unsigned x = w ^ 0x80808080u;
    const unsigned a = __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u);  // bytes u0, 0x64, u1, 0x64
    const unsigned b = __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u);  // bytes u2, 0x64, u3, 0x64
    const f16x2 bias = {(_Float16)1152.0f, (_Float16)1152.0f};
    return u32x2{__builtin_bit_cast(unsigned, __builtin_bit_cast(f16x2, a) - bias),
                 __builtin_bit_cast(unsigned, __builtin_bit_cast(f16x2, b) - bias)};
}

}  // namespace
