// What the kernels of the 8-bit key/value cache share: arguments, the rules that keep offsets, lengths and page
// numbers inside their tensors, and the codes' way into f16.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "../../include/decisive_b200.h"
#include "common.cuh"

namespace db {

constexpr int KV8_D = 128, KV8_BLK = DB_KV8_BLOCK;

struct Kv8Args {
    db_kv8_cache c;
    const int32_t* lengths;  // [items] tokens cached before this call's rows
    const int32_t* cu;       // [items + 1] rows of the items, or null: max_rows each
    int items, rows, max_rows;
    int* error;
};

// Item b: rows [start, start + count) of this call, `len` tokens cached before them; `cut` more rows are not taken (past
// max_rows, or past the table).  Offsets and lengths outside the tensors are brought back inside, and that and cut rows are
// noted in the error word.
__device__ __forceinline__ void item_of(const Kv8Args& a, int b, int& start, int& count, int& len, int& cut) {
    int rows = a.max_rows;
    if (a.cu) {
        start = min(max(a.cu[b], 0), a.rows);
        rows = min(max(a.cu[b + 1], start), a.rows) - start;
    } else {
        start = b * a.max_rows;
    }
    const int64_t most = (int64_t)a.c.table_width * KV8_BLK;
    const int given = a.lengths[b];
    count = min(rows, a.max_rows);
    len = given;
    if (given < 0 || (int64_t)given + count > most) {
        len = given < 0 ? 0 : (int)min((int64_t)given, most);
        count = (int)min((int64_t)count, most - len);
    }
    cut = rows - count;
    if ((given != len || cut) && a.error && threadIdx.x == 0) atomicOr(a.error, DB_DEV_ERR_SHAPE);
}
__device__ __forceinline__ void item_of(const Kv8Args& a, int b, int& start, int& count, int& len) {
    int cut;
    item_of(a, b, start, count, len, cut);
}

// The page that holds block i of item b, or -1 (noted in the error word) where the table names none.
__device__ __forceinline__ int page_of(const Kv8Args& a, int b, int i) {
    const int p = i < a.c.table_width ? a.c.page_table[(int64_t)b * a.c.table_width + i] : -1;
    if ((unsigned)p < (unsigned)a.c.pages) return p;
    if (a.error && (threadIdx.x & 31) == 0) atomicOr(a.error, DB_DEV_ERR_SHAPE);
    return -1;
}

__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ float from_bits(uint32_t b) {
    const unsigned short h = (unsigned short)b;
    return to_f32(*reinterpret_cast<const T*>(&h));
}

// 2^x on the special-function unit
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Four int8 codes as two pairs of f16, exactly, by the common technique of putting bits under a fixed exponent: the bytes
// become the low bits of 1024 + (code + 128).
__device__ __forceinline__ void codes_to_f16(uint32_t c, uint32_t& lo, uint32_t& hi) {
    c ^= 0x80808080u;
    const uint32_t l = __byte_perm(c, 0x64646464u, 0x4140), h = __byte_perm(c, 0x64646464u, 0x4342);
    const __half2 off = __half2half2(__ushort_as_half(0x6480));  // 1152
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&l), off);
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&h), off);
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float x, float y);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
}

struct AttnArgs {
    Kv8Args kv;
    const void* q;
    int64_t ldq;
    void* out;
    int64_t ldo;
    int group;     // query heads per kv head
    float factor;  // scale * log2 e
    float* parts;  // decode: partial results, see kv8_decode_kernel
};

// Item b's cut rows are 0 in the output: its query heads `first` .. + heads - 1, by all threads of a CTA.
template <typename T>
__device__ __forceinline__ void zero_cut_rows(const AttnArgs& a, int b, int first, int heads) {
    int start, count, len, cut;
    item_of(a.kv, b, start, count, len, cut);
    T* out = static_cast<T*>(a.out) + (int64_t)(start + count) * a.ldo + (int64_t)first * KV8_D;
    const int pieces = heads * (KV8_D / 8);
    for (int64_t i = threadIdx.x; i < (int64_t)cut * pieces; i += blockDim.x)
        *reinterpret_cast<uint4*>(out + i / pieces * a.ldo + i % pieces * 8) = make_uint4(0, 0, 0, 0);
}

// Many query rows (kv8_rows.cu).
template <typename T>
cudaError_t kv8_rows_attention(const AttnArgs& a, cudaStream_t stream);

}  // namespace db
