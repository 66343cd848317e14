// The 8-bit paged key/value cache (db_kv8_append, db_kv8_read) and the attention that reads it
// (db_kv8_attention).
//
// A sequence's tokens lie in blocks of 64.  A full block is one page of int8 codes per kv head with
// one f32 scale for its keys and one for its values: scale = max(max|x| * (1 / 127), FLT_MIN), code =
// round-half-even(x / scale).  The block that is still open is kept in 16 bits (the tail) and is
// quantised once, when its last token comes, so the codes do not depend on how the tokens were
// split over appends.  Keys are stored [64 tokens, 128], values [128, 64 tokens]: both are then
// read along the axis that their product sums over, 16 bytes at a time and without a transpose.
#include <cuda_bf16.h>
#include <float.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "../../include/decisive_b200.h"
#include "capi_internal.h"
#include "common.cuh"
#include "kernels.h"
#include "kv8.cuh"

namespace db {
namespace {

constexpr int D = KV8_D, BLK = KV8_BLK;

// ------------------------------------------------------------------ append
constexpr int APPEND_THREADS = 256;
constexpr int V_PITCH = D + 2;  // elements: rows of the value tile start on different banks

// One CTA per touched block, kv head and item.  Its 64 x 128 keys and values are gathered from the
// tail and the new rows; a full block is quantised into its page, an open one keeps its new rows in
// the tail.  The first block's CTA also writes the tail of the last block, because the two use the
// same slots and it is the one that still reads them.  HBM bound; for one token it is launch
// latency, and only a block that fills up does more than copy 512 bytes.  B200, 4 items of 1024 new tokens, 8 kv heads:
// 18 us; one token of one item: 4 us.
template <typename T>
__global__ void __launch_bounds__(APPEND_THREADS)
    kv8_append_kernel(Kv8Args a, const T* __restrict__ k, int64_t ldk, const T* __restrict__ v, int64_t ldv) {
    __shared__ uint32_t largest[2];
    __shared__ __align__(16) T vt[BLK * V_PITCH];
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, h = blockIdx.y, b = blockIdx.z, Hk = a.c.kv_heads;
    int start, count, len;
    item_of(a, b, start, count, len);
    const int first = len / BLK, block = first + blockIdx.x, total = len + count;
    if (count <= 0 || (int64_t)block * BLK >= total) return;
    const bool full = (block + 1) * BLK <= total;
    T* k_tail = static_cast<T*>(a.c.k_tail) + ((int64_t)b * Hk + h) * BLK * D;
    T* v_tail = static_cast<T*>(a.c.v_tail) + ((int64_t)b * Hk + h) * D * BLK;
    const T* krow = k + (int64_t)start * ldk + h * D;
    const T* vrow = v + (int64_t)start * ldv + h * D;

    // rows of block `w` from position max(len, 64 w) on, into the tail
    auto keep = [&](int w) {
        const int p0 = max(len, w * BLK), n = total - p0;
        for (int i = tid; i < n * (D / 8); i += APPEND_THREADS) {
            const int r = i / (D / 8), c = i % (D / 8) * 8, p = p0 + r;
            *reinterpret_cast<uint4*>(k_tail + (p % BLK) * D + c) =
                *reinterpret_cast<const uint4*>(krow + (int64_t)(p - len) * ldk + c);
        }
        // values: 8 features of a token per load, neighbouring lanes neighbouring tokens
        uint4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = (tid + i * APPEND_THREADS) % BLK, c = (tid + i * APPEND_THREADS) / BLK * 8;
            if (r < n) x[i] = *reinterpret_cast<const uint4*>(vrow + (int64_t)(p0 + r - len) * ldv + c);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = (tid + i * APPEND_THREADS) % BLK, c = (tid + i * APPEND_THREADS) / BLK * 8;
            const T* y = reinterpret_cast<const T*>(&x[i]);
            if (r < n)
#pragma unroll
                for (int j = 0; j < 8; ++j) v_tail[(c + j) * BLK + (p0 + r) % BLK] = y[j];
        }
    };
    if (!full) {
        // an open block after the first one is left to the first block's CTA
        if (blockIdx.x == 0) keep(block);
        return;
    }

    if (tid < 2) largest[tid] = 0;
    const int kept = blockIdx.x == 0 ? len % BLK : 0;  // tokens of this block that are in the tail
    uint4 key[4];
    uint32_t kmax = 0, vmax = 0;
    auto most = [](uint32_t& m, const uint4& r) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) m = max(m, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int e = tid + i * APPEND_THREADS, r = e / (D / 8), c = e % (D / 8) * 8;
        const int64_t src = (int64_t)block * BLK + r - len;
        if (r < kept) {
            key[i] = *reinterpret_cast<const uint4*>(k_tail + r * D + c);
        } else {
            key[i] = *reinterpret_cast<const uint4*>(krow + src * ldk + c);
            const uint4 x = *reinterpret_cast<const uint4*>(vrow + src * ldv + c);
            most(vmax, x);
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) *reinterpret_cast<uint32_t*>(&vt[r * V_PITCH + c + 2 * j]) = w[j];
        }
        most(kmax, key[i]);
    }
    if (kept)
        for (int e = tid; e < D * BLK / 8; e += APPEND_THREADS) {
            // (slots past the kept ones hold older tokens)
            const int c = e % D, r0 = e / D * 8;
            const uint4 x = *reinterpret_cast<const uint4*>(v_tail + c * BLK + r0);
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const unsigned short u = (unsigned short)(w[j >> 1] >> (16 * (j & 1)));
                if (r0 + j < kept) {
                    vmax = max(vmax, (uint32_t)u & 0x7fffu);
                    vt[(r0 + j) * V_PITCH + c] = *reinterpret_cast<const T*>(&u);
                }
            }
        }
    __syncthreads();
    kmax = __reduce_max_sync(0xffffffffu, kmax);
    vmax = __reduce_max_sync(0xffffffffu, vmax);
    if ((tid & 31) == 0) {
        atomicMax(&largest[0], kmax);
        atomicMax(&largest[1], vmax);
    }
    __syncthreads();
    const int page = page_of(a, b, block);
    if (page >= 0) {
        const float ka = from_bits<T>(largest[0]), va = from_bits<T>(largest[1]);
        // a block with a NaN or an infinity reads as NaN as a whole (scale NaN, codes 0)
        const float ks = isfinite(ka) ? fmaxf(__fmul_rn(ka, 1.f / 127.f), FLT_MIN) : NAN;
        const float vs = isfinite(va) ? fmaxf(__fmul_rn(va, 1.f / 127.f), FLT_MIN) : NAN;
        const int64_t ph = (int64_t)page * Hk + h;
        if (tid == 0) {
            a.c.k_scales[ph] = ks;
            a.c.v_scales[ph] = vs;
        }
        // round half even (x / s): the product with 1 / s (off by 2^-16 at most) decides unless it lies near a half.  Rounding by
        // a large addend is a common technique: 1.5 x 2^23 + code has the code's two's complement in its low byte, and |x / s|
        // never passes 127.
        const float ki = __fdiv_rn(1.f, ks), vi = __fdiv_rn(1.f, vs);
        constexpr float MAGIC = 12582912.f;
        auto four = [](const float (&x)[4], float s, float inverse) {
            uint32_t r[4];
            bool near = false;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float y = fmaf(x[j], inverse, MAGIC), left = fmaf(x[j], inverse, -(y - MAGIC));
                near |= !(fabsf(left) < 0.4999f);
                r[j] = __float_as_uint(y);
            }
            if (near) {
#pragma unroll 1
                for (int j = 0; j < 4; ++j) {
                    const float v = j == 0 ? x[0] : j == 1 ? x[1] : j == 2 ? x[2] : x[3];
                    const uint32_t y = s == s ? __float_as_uint(rintf(__fdiv_rn(v, s)) + MAGIC) : 0u;
                    r[0] = j == 0 ? y : r[0], r[1] = j == 1 ? y : r[1], r[2] = j == 2 ? y : r[2], r[3] = j == 3 ? y : r[3];
                }
            }
            return __byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410);
        };
        int8_t* kp = a.c.k_codes + ph * BLK * D;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = tid + i * APPEND_THREADS;
            const float x[4] = {from_bits<T>(key[i].x & 0xffffu), from_bits<T>(key[i].x >> 16), from_bits<T>(key[i].y & 0xffffu),
                                from_bits<T>(key[i].y >> 16)};
            const float y[4] = {from_bits<T>(key[i].z & 0xffffu), from_bits<T>(key[i].z >> 16), from_bits<T>(key[i].w & 0xffffu),
                                from_bits<T>(key[i].w >> 16)};
            *reinterpret_cast<uint2*>(kp + (int64_t)e * 8) = make_uint2(four(x, ks, ki), four(y, ks, ki));
        }
        int8_t* vp = a.c.v_codes + ph * D * BLK;
#pragma unroll
        for (int i = 0; i < D * BLK / 16 / APPEND_THREADS; ++i) {
            const int e = tid + i * APPEND_THREADS, c = e % D, r0 = e / D * 16;  // value feature c, tokens r0 .. r0 + 15
            uint32_t o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float x[4] = {to_f32(vt[(r0 + 4 * j) * V_PITCH + c]), to_f32(vt[(r0 + 4 * j + 1) * V_PITCH + c]),
                                    to_f32(vt[(r0 + 4 * j + 2) * V_PITCH + c]), to_f32(vt[(r0 + 4 * j + 3) * V_PITCH + c])};
                o[j] = four(x, vs, vi);
            }
            *reinterpret_cast<uint4*>(vp + c * BLK + r0) = make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
    const int last = total / BLK;  // the block that stays open
    if (blockIdx.x == 0 && last > first && total % BLK) keep(last);
}

// ------------------------------------------------------------------ read back
// The cached values of tokens 0 .. max_keys - 1 in f32 (0 past an item's length).  One CTA per block, kv head and
// keys or values; HBM bound.  16-byte loads and stores; the values turn in shared memory.  B200, 4 items of some 1200
// tokens, 8 kv heads: 14 us (48 MB, most of it the f32 output, which stays in the L2 cache at that size).
constexpr int READ_THREADS = 256, READ_PITCH = D + 4;

template <typename T>
__global__ void __launch_bounds__(READ_THREADS)
    kv8_read_kernel(Kv8Args a, int64_t max_keys, float* __restrict__ k, float* __restrict__ v) {
    __shared__ __align__(16) float tile[BLK * READ_PITCH];
    pdl_wait();
    const int tid = threadIdx.x, which = blockIdx.x & 1, block = blockIdx.x >> 1, h = blockIdx.y, b = blockIdx.z;
    const int Hk = a.c.kv_heads;
    int start, count, len;
    item_of(a, b, start, count, len);
    const int n = (int)min((int64_t)BLK, max_keys - (int64_t)block * BLK);
    const bool full = (int64_t)(block + 1) * BLK <= len;
    const int inside = min(max(len - block * BLK, 0), BLK);
    const int page = full ? page_of(a, b, block) : -1;
    const int64_t ph = (int64_t)page * Hk + h, tail = ((int64_t)b * Hk + h) * BLK * D;
    // 16 values at a time: of one token for keys (row r, features c ..), of one feature for values
    for (int e = tid; e < BLK * D / 16; e += READ_THREADS) {
        const int r = which ? e / D * 16 : e / (D / 16), c = which ? e % D : e % (D / 16) * 16;
        const int64_t at = which ? (int64_t)c * BLK + r : (int64_t)r * D + c;
        float x[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = 0.f;
        if (page >= 0) {
            const uint4 w = *reinterpret_cast<const uint4*>((which ? a.c.v_codes : a.c.k_codes) + ph * BLK * D + at);
            const float scale = (which ? a.c.v_scales : a.c.k_scales)[ph];
            const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int j = 0; j < 16; ++j)
                x[j] = __fmul_rn((float)(int)(int8_t)(q[j >> 2] >> (8 * (j & 3))), scale);
        } else if (!full && (which || r < inside)) {
            const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(which ? a.c.v_tail : a.c.k_tail) + tail + at);
            const uint4 w0 = src[0], w1 = src[1];
            const uint32_t q[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (!which || r + j < inside) x[j] = from_bits<T>((q[j >> 1] >> (16 * (j & 1))) & 0xffffu);
        }
        if (which) {
#pragma unroll
            for (int j = 0; j < 16; ++j) tile[(r + j) * READ_PITCH + c] = x[j];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *reinterpret_cast<float4*>(&tile[r * READ_PITCH + c + 4 * j]) =
                    make_float4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
        }
    }
    __syncthreads();
    float* out = (which ? v : k) + (((int64_t)b * max_keys + (int64_t)block * BLK) * Hk + h) * D;
    for (int e = tid; e < n * (D / 4); e += READ_THREADS) {
        const int r = e / (D / 4), c = e % (D / 4) * 4;
        __stcs(reinterpret_cast<float4*>(out + (int64_t)r * Hk * D + c),
               *reinterpret_cast<const float4*>(&tile[r * READ_PITCH + c]));
    }
}

// ------------------------------------------------------------------ attention
// mma.sync m16n8k16 with f32 accumulators: D [16, 8] += A [16, 16] B [16, 8].
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The 8 x 8 matrix of 16-bit values that a warp holds, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// Scores and the context are formed transposed, S^T = K Q^T and O^T = V^T P^T, so that the codes are
// the wide operand (16 keys or 16 value features of an MMA) and 8 query rows the narrow one: a single
// token's 4 or 8 heads fill it.  Row n of a kv head's tile is query (token n / group, head n % group).
//
// Every lane reads 16 codes in one load and they are exactly what its MMA fragments need, because
// the order of a product's sum is free: within a 64-wide half of a key, k step s of the fragment takes
// bytes 4s..4s+3 of each lane's 16; and key 16 (r >> 1) + 4 s + 2 half + (r & 1) sits in row r of
// half `half` of score tile s, which makes P^T's fragment the four bytes 4s..4s+3 of each 16 of V^T.
// Codes become f16 exactly; q is scaled by a power of two per row into f16 (bf16 has fewer bits
// and more range), so the scores' product rounds neither operand.  P enters its product as two f16 parts, 22 bits (one
// f16 would change one bf16 output in 15 and is as large a rounding as an f16 output's own), as 2^15 P, so that f16's
// subnormals begin 2^-29 below the largest: thousands of weak keys beside one strong one without a value still add up.  Its
// sum is taken from the f32 values.  A block's own context is scaled by its value scale when it joins the running one, in f32.
//
// The tile of 8 NT query rows that a warp works on, with its running maxima and sums (log2 domain; column
// 2 t + j of n tile n in [n][j], equal in the 8 lanes g) and its context (feature 16 d + 8 (j >> 1) + g).
constexpr float LIFT = 15.f, DROP = 3.0517578e-5f;  // 2^-15

template <typename T, int NT>
struct Tile {
    // query fragments, k step 4 c + s: in registers, or for more rows in shared memory ([NT][8][32], the warp's own)
    uint2 qf[NT == 1 ? 8 : 1];
    uint2* qs;
    float factor[NT][2];   // scale * log2 e / the row's power of two
    int limit[NT][2];      // last key that a column's row sees; -1: none
    int first_limit;       // of the tile's first row
    bool ragged;           // rows past the item's end
    float m[NT][2], l[NT][2];
    float O[8][NT][4];
    // where the rows are
    const T* q;
    int row0, rows, group;
    int64_t ldq;
    float plain;           // scale * log2 e

    __device__ uint2 query(int n, int step) const {
        if constexpr (NT == 1) return qf[step];
        return qs[(n * 8 + step) * 32 + (threadIdx.x & 31)];
    }
    __device__ const T* row_at(int r) const { return q + (int64_t)(r / group) * ldq + (int64_t)(r % group) * D; }

    // q: the item's first row at the kv head's first query head; the tile starts at row r0 of `all`
    __device__ void open(uint2* shared, const T* base, int64_t ld, int r0, int all, int len, int grp, float fac) {
        qs = shared;
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        q = base, ldq = ld, row0 = r0, rows = all, group = grp, plain = fac;
        first_limit = len + r0 / grp;
        ragged = r0 + 8 * NT > all;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = r0 + n * 8 + g;
            uint32_t w[16];
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint4 x = make_uint4(0, 0, 0, 0);
                    if (r < all) x = *reinterpret_cast<const uint4*>(row_at(r) + 64 * c + 16 * t + 8 * i);
                    w[8 * c + 4 * i] = x.x, w[8 * c + 4 * i + 1] = x.y, w[8 * c + 4 * i + 2] = x.z, w[8 * c + 4 * i + 3] = x.w;
                }
            // to [2^8, 2^9) at the row's largest value
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) top = max(top, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float big = from_bits<T>(top);
            const int e = (int)(__float_as_uint(big) >> 23) - 127;
            const int k = big > 0.f && e < 128 ? min(max(8 - e, -126), 126) : 0;
            const float up = __uint_as_float((uint32_t)(127 + k) << 23), back = __uint_as_float((uint32_t)(127 - k) << 23);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                uint2 x;
                x.x = pack2<__half>(from_bits<T>(w[2 * i] & 0xffffu) * up, from_bits<T>(w[2 * i] >> 16) * up);
                x.y = pack2<__half>(from_bits<T>(w[2 * i + 1] & 0xffffu) * up, from_bits<T>(w[2 * i + 1] >> 16) * up);
                if constexpr (NT == 1)
                    qf[i] = x;
                else
                    qs[(n * 8 + i) * 32 + lane] = x;
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                factor[n][j] = fac * __shfl_sync(0xffffffffu, back, 4 * (2 * t + j));
                const int rr = r0 + n * 8 + 2 * t + j;
                limit[n][j] = rr < all ? len + rr / grp : -1;
                m[n][j] = -INFINITY;
                l[n][j] = 0.f;
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) O[i][n][j] = 0.f;
    }

    // S^T of the block at key `base` is in s (16 keys per tile): softmax step; leaves 2^lift P in f32 in s (drop: 2^-lift)
    // and the factors of the running context in alpha
    __device__ void soften(float (&s)[4][NT][4], const float (&f)[NT][2], int base, float (&alpha)[NT][2], float lift, float drop) {
        const int lane = threadIdx.x & 31, g = lane >> 2;
        const bool masked = base + BLK - 1 > first_limit || ragged;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float x = s[i][n][j] * f[n][j & 1];
                    if (masked) {
                        const int key = base + 16 * (g >> 1) + 4 * i + 2 * (j >> 1) + (g & 1);
                        x = key <= limit[n][j & 1] ? x : -INFINITY;
                    }
                    s[i][n][j] = x;
                    top[j & 1] = fmaxf(top[j & 1], x);
                }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int o = 4; o < 32; o *= 2) top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], o));
                const float now = fmaxf(m[n][j], top[j]);
                const float at = now == -INFINITY ? 0.f : now;
                alpha[n][j] = ex2(m[n][j] - at);
                m[n][j] = now;
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const float p = ex2((s[i][n][2 * half + j] - at) + lift);  // (large scores: the difference first)
                        s[i][n][2 * half + j] = p;
                        sum += p;
                    }
                l[n][j] = fmaf(sum, drop, l[n][j] * alpha[n][j]);
            }
        }
    }

    // a lane's share of a block's key codes: score tile, row half, 64-wide half of the key
    __device__ static void load_keys(uint4 (&kc)[4][2][2], const int8_t* kp) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int c = 0; c < 2; ++c)
                    kc[s][r][c] = __ldcs(reinterpret_cast<const uint4*>(
                        kp + (16 * (g >> 1) + 4 * s + 2 * r + (g & 1)) * D + 64 * c + 16 * t));
    }

    // one full block: 64 keys' and values' codes of one head.  Its values are on their way while the scores are
    // formed, and the next block's keys (after: null for none) while the context is: a warp always has 8 KB of
    // loads in flight.
    __device__ void block(uint4 (&kc)[4][2][2], const int8_t* vp, float ks, float vs, int base, const int8_t* after) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        constexpr bool AHEAD = NT == 1;  // (more rows leave no registers for it)
        uint4 vc[AHEAD ? 8 : 1][2];
        if constexpr (AHEAD)
#pragma unroll
            for (int d = 0; d < 8; ++d)
#pragma unroll
                for (int r = 0; r < 2; ++r)
                    vc[d][r] = __ldcs(reinterpret_cast<const uint4*>(vp + (16 * d + 8 * r + g) * BLK + 16 * t));
        float s[4][NT][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[i][n][j] = 0.f;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const uint32_t lo[4] = {kc[i][0][c].x, kc[i][0][c].y, kc[i][0][c].z, kc[i][0][c].w};
                const uint32_t hi[4] = {kc[i][1][c].x, kc[i][1][c].y, kc[i][1][c].z, kc[i][1][c].w};
#pragma unroll
                for (int st = 0; st < 4; ++st) {
                    uint32_t f[4];
                    codes_to_f16(lo[st], f[0], f[2]);
                    codes_to_f16(hi[st], f[1], f[3]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const uint2 q2 = query(n, 4 * c + st);
                        mma16(s[i][n], f, q2.x, q2.y, __half());
                    }
                }
            }
        }
        if (after) load_keys(kc, after);
        const bool lifted = vs >= 1e-30f;  // (the value scale takes the factor back, as long as it stays a normal number)
        const float drop = lifted ? DROP : 1.f, back = vs * drop;
        float alpha[NT][2], scaled[NT][2], vf[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                scaled[n][j] = factor[n][j] * ks;
                vf[n][j] = limit[n][j] >= base ? back : 0.f;  // a block that a row does not see must not reach it (0 x NaN)
            }
        soften(s, scaled, base, alpha, lifted ? LIFT : 0.f, drop);
        uint32_t p[NT][4][2], rest[NT][4][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const float x = s[i][n][2 * half], y = s[i][n][2 * half + 1];
                    const uint32_t hi = pack2<__half>(x, y);
                    p[n][i][half] = transpose8(hi);
                    rest[n][i][half] =
                        transpose8(pack2<__half>(x - from_bits<__half>(hi & 0xffffu), y - from_bits<__half>(hi >> 16)));
                }
#pragma unroll
        for (int d = 0; d < 8; ++d) {
            uint4 v0, v1;
            if constexpr (AHEAD) {
                v0 = vc[d][0], v1 = vc[d][1];
            } else {
                v0 = __ldcs(reinterpret_cast<const uint4*>(vp + (16 * d + g) * BLK + 16 * t));
                v1 = __ldcs(reinterpret_cast<const uint4*>(vp + (16 * d + 8 + g) * BLK + 16 * t));
            }
            const uint32_t lo[4] = {v0.x, v0.y, v0.z, v0.w}, hi[4] = {v1.x, v1.y, v1.z, v1.w};
            float o[NT][4] = {};
#pragma unroll
            for (int st = 0; st < 4; ++st) {
                uint32_t f[4];
                codes_to_f16(lo[st], f[0], f[2]);
                codes_to_f16(hi[st], f[1], f[3]);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    mma16(o[n], f, p[n][st][0], p[n][st][1], __half());
                    mma16(o[n], f, rest[n][st][0], rest[n][st][1], __half());
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) O[d][n][j] = fmaf(o[n][j], vf[n][j & 1], O[d][n][j] * alpha[n][j & 1]);
        }
    }

    // the open block, in 16 bits: the same walk on its own type, rolled up (it is one of many blocks, and code
    // that runs once costs its fetching); `inside` tokens of it are there
    __device__ void tail(const T* kt, const T* vt, int inside, int base) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        float s[4][NT][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[i][n][j] = 0.f;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {  // 8 of each lane's 16 dims of a half
            const int at = 64 * (c >> 1) + 16 * t + 8 * (c & 1);
            uint4 qr[NT], kr[4][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) qr[n] = *reinterpret_cast<const uint4*>(row_at(min(row0 + n * 8 + g, rows - 1)) + at);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int r = 0; r < 2; ++r)
                    kr[i][r] = *reinterpret_cast<const uint4*>(kt + (16 * (g >> 1) + 4 * i + 2 * r + (g & 1)) * D + at);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t f0[4] = {kr[i][0].x, kr[i][1].x, kr[i][0].y, kr[i][1].y};
                const uint32_t f1[4] = {kr[i][0].z, kr[i][1].z, kr[i][0].w, kr[i][1].w};
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    mma16(s[i][n], f0, qr[n].x, qr[n].y, T());
                    mma16(s[i][n], f1, qr[n].z, qr[n].w, T());
                }
            }
        }
        constexpr int PARTS = std::is_same<T, __half>::value ? 2 : 3;
        constexpr float drop = PARTS == 2 ? DROP : 1.f;
        float alpha[NT][2], unscaled[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) unscaled[n][0] = unscaled[n][1] = plain;
        soften(s, unscaled, base, alpha, PARTS == 2 ? LIFT : 0.f, drop);
        // P in parts of the tail's type: two of f16 hold 22 bits, three of bf16 24 (which has no need of the lift)
        uint32_t p[PARTS][NT][4][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    float x = s[i][n][2 * half], y = s[i][n][2 * half + 1];
#pragma unroll
                    for (int k = 0; k < PARTS; ++k) {
                        const uint32_t part = pack2<T>(x, y);
                        p[k][n][i][half] = transpose8(part);
                        x -= from_bits<T>(part & 0xffffu);
                        y -= from_bits<T>(part >> 16);
                    }
                }
        constexpr int BATCH = NT == 1 ? 2 : 1;  // feature tiles whose values are loaded together
#pragma unroll 1
        for (int d0 = 0; d0 < 8; d0 += BATCH) {
            uint32_t f[BATCH][2][8];
#pragma unroll
            for (int d = 0; d < BATCH; ++d)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const uint4* src = reinterpret_cast<const uint4*>(vt + (16 * (d0 + d) + 8 * r + g) * BLK + 16 * t);
                    const uint4 x = src[0], y = src[1];
                    f[d][r][0] = x.x, f[d][r][1] = x.y, f[d][r][2] = x.z, f[d][r][3] = x.w;
                    f[d][r][4] = y.x, f[d][r][5] = y.y, f[d][r][6] = y.z, f[d][r][7] = y.w;
                }
            float o[BATCH][NT][4];
            bool odd = false;  // a NaN or an infinity among the values
#pragma unroll
            for (int d = 0; d < BATCH; ++d) {
#pragma unroll
                for (int r = 0; r < 2; ++r)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        // slots that hold no token yet, and what is not finite, stay out of the product
                        constexpr uint32_t INF = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
                        const int key = 16 * t + 2 * e;
                        uint32_t lo = key < inside ? f[d][r][e] & 0xffffu : 0, hi = key + 1 < inside ? f[d][r][e] >> 16 : 0;
                        const bool bl = (lo & INF) == INF, bh = (hi & INF) == INF;
                        odd |= bl | bh;
                        f[d][r][e] = (bl ? 0 : lo) | (bh ? 0 : hi) << 16;
                    }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[d][n][j] = 0.f;
#pragma unroll
                for (int st = 0; st < 4; ++st) {
                    const uint32_t fa[4] = {f[d][0][2 * st], f[d][1][2 * st], f[d][0][2 * st + 1], f[d][1][2 * st + 1]};
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int k = 0; k < PARTS; ++k) mma16(o[d][n], fa, p[k][n][st][0], p[k][n][st][1], T());
                }
            }
            if (__any_sync(0xffffffffu, odd)) {
                // such a value reaches the rows that see its key, and no other
#pragma unroll
                for (int d = 0; d < BATCH; ++d)
#pragma unroll
                    for (int r = 0; r < 2; ++r)
#pragma unroll 1
                        for (int key = 0; key < min(inside, BLK); ++key) {
                            const float x = to_f32(vt[(16 * (d0 + d) + 8 * r + g) * BLK + key]);
                            if (isfinite(x)) continue;
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int j = 0; j < 2; ++j)
                                    if (base + key <= limit[n][j]) o[d][n][2 * r + j] += x;
                        }
            }
#pragma unroll
            for (int d = 0; d < 8; ++d)
                if (d >= d0 && d < d0 + BATCH)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            O[d][n][j] = fmaf(O[d][n][j], alpha[n][j & 1], o[d % BATCH][n][j] * drop);
        }
    }

    // l over the lanes that share a column
    __device__ void close() {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int o = 4; o < 32; o *= 2) l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], o);
    }

    // the finished rows; out: the item's first row at the kv head's first query head
    __device__ void write(T* out, int64_t ldo) const {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float i0 = l[n][0] == 0.f ? 0.f : 1.f / l[n][0], i1 = l[n][1] == 0.f ? 0.f : 1.f / l[n][1];
            const int r = row0 + n * 8 + g;
            T* dst = out + (int64_t)(r / group) * ldo + (int64_t)(r % group) * D + 2 * t;
#pragma unroll
            for (int d = 0; d < 8; ++d)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint32_t w = transpose8(pack2<T>(O[d][n][2 * half] * i0, O[d][n][2 * half + 1] * i1));
                    if (r < rows) *reinterpret_cast<uint32_t*>(dst + 16 * d + 8 * half) = w;
                }
        }
    }
};

// ------------------------------------------------------------------ few rows: the blocks dealt out evenly
// All blocks of all items and kv heads form one row of units, (item, head, block), that is cut into equal runs,
// one per warp; a tile's start counts TILE_COST units more (its queries, its open block, its end: short sequences
// cost more than their blocks); so sequences of any lengths keep every warp busy alike, and no warp waits for another.  A
// warp writes the tiles whose blocks it has all; of a tile that it shares it leaves (O, m, l) in its slot
// 0 (the tile began before its run) or 1 (it goes on after it), and kv8_join_kernel adds the slots up in order.
// Bound by HBM and by the issue of what turns codes into products (P's second part, without which bf16 took 90 us where it
// takes 101): the codes are read once, straight into the fragments' registers.  B200, 32 / 8 heads, this kernel alone, f16
// and bf16 alike: 4 items of 60 to 65 thousand keys 101 us (5.2 TB/s, 80% of the copy's rate), 64 items of 1 to 8191 keys
// 111 us (4.6 TB/s); one item of 544 keys 14 us and 12 us for the join.
constexpr int DECODE_WARPS = 4, TILE_COST = 2;
__host__ __device__ constexpr int part_floats(int nt) { return (32 + 4) * nt * 32; }  // O and m, l in the lanes' order

// Where a unit lies.  sums[i]: units (of one head) of the items before chunk i of `per` items.
struct Units {
    int64_t total;  // units of all items, one head
    int per;
    bool cut;       // some item has rows that are cut off
};
// Blocks that item b's rows see.
__device__ __forceinline__ int blocks_of(int count, int len) { return count > 0 ? (len + count - 1) / BLK + 1 : 0; }
__device__ __forceinline__ int item_blocks(const Kv8Args& a, int b, int& start, int& count, int& len) {
    item_of(a, b, start, count, len);
    return blocks_of(count, len);
}
__device__ __forceinline__ int item_units(const Kv8Args& a, int b, int& start, int& count, int& len) {
    const int n = item_blocks(a, b, start, count, len);
    return n ? n + TILE_COST : 0;
}
template <int THREADS>
__device__ Units count_units(const Kv8Args& a, int64_t* sums) {  // sums: [THREADS + 1] in shared memory
    __shared__ int64_t warp_sum[THREADS / 32];
    const int tid = threadIdx.x, lane = tid & 31;
    Units u;
    u.per = (a.items + THREADS - 1) / THREADS;
    int64_t mine = 0;
    int cut = 0;
    for (int b = tid * u.per; b < min((tid + 1) * u.per, a.items); ++b) {
        int s, c, l, off;
        item_of(a, b, s, c, l, off);
        const int n = blocks_of(c, l);
        mine += n ? n + TILE_COST : 0;
        cut |= off;
    }
    int64_t run = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const int64_t y = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += y;
    }
    if (lane == 31) warp_sum[tid >> 5] = run;
    __syncthreads();
    for (int w = 0; w < (tid >> 5); ++w) run += warp_sum[w];
    sums[tid + 1] = run;
    if (tid == 0) sums[0] = 0;
    u.cut = __syncthreads_or(cut);
    u.total = sums[THREADS];
    return u;
}
// Item of unit x (of one head; x < total) and the units before it.
template <int THREADS>
__device__ int find_item(const Kv8Args& a, const int64_t* sums, const Units& u, int64_t x, int64_t& before) {
    int lo = 0, hi = THREADS - 1;  // last chunk whose sum is <= x
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (sums[mid] <= x) lo = mid; else hi = mid - 1;
    }
    int b = lo * u.per;
    before = sums[lo];
    for (;; ++b) {
        int s, c, l;
        const int n = item_units(a, b, s, c, l);
        if (x < before + n || b == a.items - 1) return b;
        before += n;
    }
}
// Units of a warp's run.
__device__ __forceinline__ int64_t run_length(int64_t units, int64_t warps) { return max((units + warps - 1) / warps, (int64_t)1); }

template <typename T, int NT>
__global__ void __launch_bounds__(32 * DECODE_WARPS, 2) kv8_decode_kernel(AttnArgs a) {
    __shared__ int64_t sums[32 * DECODE_WARPS + 1];
    __shared__ uint2 queries[NT == 1 ? 1 : DECODE_WARPS][NT == 1 ? 1 : NT * 8 * 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, Hk = a.kv.c.kv_heads;
    pdl_wait();
    pdl_trigger();
    const Units units = count_units<32 * DECODE_WARPS>(a.kv, sums);
    for (int b = blockIdx.x; units.cut && b < a.kv.items; b += gridDim.x) zero_cut_rows<T>(a, b, 0, Hk * a.group);
    const int64_t all = units.total * Hk, per = run_length(all, (int64_t)gridDim.x * DECODE_WARPS);
    const int64_t w = (int64_t)blockIdx.x * DECODE_WARPS + warp, begin = w * per, end = min(begin + per, all);
    // units run (item, head, block): the items before x units of one head take x Hk units
    int64_t u = begin;
    while (u < end) {
        int64_t before;
        const int b = find_item<32 * DECODE_WARPS>(a.kv, sums, units, u / Hk, before);
        int start, count, len;
        const int n = item_blocks(a.kv, b, start, count, len);
        const int64_t inner = u - before * Hk;
        int h = (int)(inner / (n + TILE_COST)), at_unit = (int)(inner % (n + TILE_COST));
        // the heads of this item, as far as the run goes
        for (; h < Hk && u < end; ++h, at_unit = 0) {
            const int until = (int)min((int64_t)n + TILE_COST, at_unit + (end - u));
            const int first = max(at_unit - TILE_COST, 0), last = max(until - TILE_COST, 0);
            u += until - at_unit;
            if (first == last) continue;  // of this tile the run has only its cost
            int i = first;
            Tile<T, NT> tile;
            tile.open(queries[NT == 1 ? 0 : warp], static_cast<const T*>(a.q) + (int64_t)start * a.ldq + (int64_t)h * a.group * D, a.ldq, 0,
                      count * a.group, len, a.group, a.factor);
            const int whole = (len + count) / BLK;
            // pages one block ahead, keys from the block before (a block without a page breaks the chain)
            const int stop = min(last, whole);
            const auto keys_of = [&](int p) { return a.kv.c.k_codes + ((int64_t)p * Hk + h) * BLK * D; };
            int page = i < stop ? page_of(a.kv, b, i) : -1;
            int next = i + 1 < stop ? page_of(a.kv, b, i + 1) : -1;
            uint4 kc[4][2][2];
            if (page >= 0) tile.load_keys(kc, keys_of(page));
            for (; i < stop; ++i) {
                const int later = i + 2 < stop ? page_of(a.kv, b, i + 2) : -1;
                if (page >= 0) {
                    const int64_t ph = (int64_t)page * Hk + h;
                    tile.block(kc, a.kv.c.v_codes + ph * BLK * D, a.kv.c.k_scales[ph], a.kv.c.v_scales[ph], i * BLK,
                               next >= 0 ? keys_of(next) : nullptr);
                } else if (next >= 0) {
                    tile.load_keys(kc, keys_of(next));
                }
                page = next, next = later;
            }
            if (last > stop) {
                const int64_t at = ((int64_t)b * Hk + h) * BLK * D;
                tile.tail(static_cast<const T*>(a.kv.c.k_tail) + at, static_cast<const T*>(a.kv.c.v_tail) + at,
                          len + count - whole * BLK, whole * BLK);
            }
            tile.close();
            if (first == 0 && last == n) {
                tile.write(static_cast<T*>(a.out) + (int64_t)start * a.ldo + (int64_t)h * a.group * D, a.ldo);
                continue;
            }
            float* part = a.parts + (2 * w + (first == 0 ? 1 : 0)) * part_floats(NT) + lane;
#pragma unroll
            for (int k = 0; k < NT; ++k) {
#pragma unroll
                for (int d = 0; d < 8; ++d)
#pragma unroll
                    for (int j = 0; j < 4; ++j) part[((k * 8 + d) * 4 + j) * 32] = tile.O[d][k][j];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    part[(32 * NT + 4 * k + j) * 32] = tile.m[k][j];
                    part[(32 * NT + 4 * k + 2 + j) * 32] = tile.l[k][j];
                }
            }
        }
    }
}

// Adds up the slots of a tile that several warps shared, in order: a CTA per kv head, item and quarter of the
// tile (value features 32 x .. + 31), a thread per value of the context in the slots' own layout.  Latency
// bound: the slots' maxima and sums are turned into weights first, then all loads are independent.
constexpr int JOIN_SLOTS = 64;  // slots at a time

template <typename T, int NT>
__global__ void __launch_bounds__(256 * NT) kv8_join_kernel(AttnArgs a, int64_t warps) {
    constexpr int ROWS = 8 * NT, THREADS = 256 * NT;
    __shared__ int64_t sums[THREADS + 1];
    __shared__ float weight[JOIN_SLOTS][ROWS], top[ROWS], total[ROWS], scale[ROWS];
    const int tid = threadIdx.x, lane = tid & 31;
    const int quarter = blockIdx.x & 3, h = blockIdx.x >> 2, b = blockIdx.y, Hk = a.kv.c.kv_heads;
    pdl_wait();
    pdl_trigger();
    const Units units = count_units<THREADS>(a.kv, sums);
    const int64_t per = run_length(units.total * Hk, warps);
    int start, count, len;
    const int n = item_blocks(a.kv, b, start, count, len);
    if (n == 0) return;
    int64_t before = sums[b / units.per];
    for (int i = b / units.per * units.per; i < b; ++i) {
        int s, c, l;
        before += item_units(a.kv, i, s, c, l);
    }
    const int64_t u0 = before * Hk + (int64_t)h * (n + TILE_COST) + TILE_COST, w0 = u0 / per, w1 = (u0 + n - 1) / per;
    if (w0 == w1) return;  // one warp had it all
    // the tile's first warp left it in slot 1, the others in slot 0
    auto slot = [&](int64_t w) { return a.parts + (2 * w + (w == w0 ? 1 : 0)) * part_floats(NT); };
    // thread: n tile, feature group 2 quarter + (0, 1), value j of the fragment, lane; its row is 8 k + 2 t + (j & 1)
    const int k = tid / 256, in = tid % 256, d = 2 * quarter + in / 128, j = in / 32 % 4;
    const int row = 8 * k + 2 * (lane & 3) + (j & 1);
    if (tid < ROWS) top[tid] = -INFINITY, total[tid] = 0.f;
    float o = 0.f;
    for (int64_t from = w0; from <= w1; from += JOIN_SLOTS) {
        const int m = (int)min((int64_t)JOIN_SLOTS, w1 - from + 1);
        __syncthreads();
        for (int e = tid; e < m * ROWS; e += THREADS) {
            const int r = e % ROWS, i = e / ROWS;
            weight[i][r] = slot(from + i)[(32 * NT + 4 * (r / 8) + (r & 1)) * 32 + (r % 8) / 2];
        }
        __syncthreads();
        if (tid < ROWS) {
            float now = top[tid];
            for (int i = 0; i < m; ++i) now = fmaxf(now, weight[i][tid]);
            scale[tid] = now == -INFINITY ? 0.f : ex2(top[tid] - now);
            top[tid] = now;
        }
        __syncthreads();
        for (int e = tid; e < m * ROWS; e += THREADS) {
            const int r = e % ROWS, i = e / ROWS;
            weight[i][r] = top[r] == -INFINITY ? 0.f : ex2(weight[i][r] - top[r]);
        }
        __syncthreads();
        if (tid < ROWS) {
            float l = total[tid] * scale[tid];
#pragma unroll 8
            for (int i = 0; i < m; ++i) l = fmaf(slot(from + i)[(32 * NT + 4 * (tid / 8) + 2 + (tid & 1)) * 32 + (tid % 8) / 2], weight[i][tid], l);
            total[tid] = l;
        }
        o *= scale[row];
#pragma unroll 16
        for (int i = 0; i < m; ++i) o = fmaf(slot(from + i)[((k * 8 + d) * 4 + j) * 32 + lane], weight[i][row], o);
    }
    __syncthreads();
    // value feature 16 d + 8 (j >> 1) + g of the row
    const float l = total[row];
    if (row < count * a.group) {
        T y;
        const float x = l == 0.f ? 0.f : o / l;
        const uint32_t two = pack2<T>(x, x);
        y = *reinterpret_cast<const T*>(&two);
        T* out = static_cast<T*>(a.out) + (int64_t)(start + row / a.group) * a.ldo + ((int64_t)h * a.group + row % a.group) * D;
        out[16 * d + 8 * (j >> 1) + (lane >> 2)] = y;
    }
}

// ------------------------------------------------------------------ launches
// n tiles of 8 rows for the dealt-out form; 0: many rows (kv8_rows.cu), which is all there is above 16.  One tile / two / many
// rows, us with the join, bf16, 8 kv heads: 64 items of 4000 keys, 4 rows per kv head 132 / 216 / 356, 8 rows 134 / 216 / 358,
// 16 rows - / 218 / 362; one item of 32000 keys, 4 rows 58 / 73 / 506, 16 rows - / 73 / 506; 4 items of 512 keys, 4 rows
// 22 / 26 / 23, 16 rows - / 26 / 23.  So rows decide: the many-row form gains 3 us on short histories and loses most of
// its time on long ones, where it has a CTA per 128 rows and kv head and does not split the keys (20 rows: 367, 510, 23 us).
int decode_tiles(int64_t rows) { return rows <= 8 ? 1 : rows <= 16 ? 2 : 0; }
// CTAs of the dealt-out form: as many as are resident at once, fewer when there are not that many blocks
int64_t decode_ctas(int64_t items, int64_t heads, int64_t max_keys) {
    const int64_t most = (int64_t)db_num_sms() * 2;
    const int64_t blocks = items * heads * ((max_keys + BLK - 1) / BLK + TILE_COST);
    return std::max<int64_t>(1, std::min(most, (blocks + DECODE_WARPS - 1) / DECODE_WARPS));
}

template <typename T, int NT>
cudaError_t launch_decode(const AttnArgs& a, int64_t max_keys, cudaStream_t stream) {
    const int64_t ctas = decode_ctas(a.kv.items, a.kv.c.kv_heads, max_keys);
    cudaError_t e = db_launch_pdl(kv8_decode_kernel<T, NT>, dim3((unsigned)ctas), dim3(32 * DECODE_WARPS), 0, stream, a);
    if (e != cudaSuccess) return e;
    return db_launch_pdl(kv8_join_kernel<T, NT>, dim3(4 * a.kv.c.kv_heads, a.kv.items), dim3(256 * NT), 0, stream, a,
                         ctas * DECODE_WARPS);
}

template <typename T>
cudaError_t attention(const AttnArgs& a, int64_t max_keys, cudaStream_t stream) {
    const int64_t rows = (int64_t)a.kv.max_rows * a.group;
    const int nt = decode_tiles(rows);
    if (nt == 1) return launch_decode<T, 1>(a, max_keys, stream);
    if (nt == 2) return launch_decode<T, 2>(a, max_keys, stream);
    return kv8_rows_attention<T>(a, stream);
}

// What every call on a cache checks; fills the arguments that they share.
int cache_args(const db_kv8_cache* c, const int32_t* lengths, const int32_t* cu, int64_t items, int64_t rows,
               int64_t max_rows, const char* what, Kv8Args* a) {
    const std::string name(what);
    if (!c || c->dtype != DB_DTYPE_F16 && c->dtype != DB_DTYPE_BF16)
        return db_fail(DB_ERR_UNSUPPORTED, "UNSUPPORTED", name + ": the open block is f16 or bf16");
    if (c->head_dim != D) return db_fail(DB_ERR_UNSUPPORTED, "UNSUPPORTED", name + ": head_dim must be 128");
    const int64_t most = (int64_t)1 << 31;
    if (items < 0 || items > 65535 || items > c->sequences || rows < 0 || rows >= most || max_rows < 0 || max_rows > rows ||
        (!cu && rows != items * max_rows) || c->kv_heads <= 0 || c->kv_heads > 65535 || c->pages < 0 ||
        c->table_width < 0 || (int64_t)c->table_width * BLK >= most - BLK)
        return db_fail(DB_ERR_INVALID_ARGUMENT, "INVALID_ARGUMENT", name + ": bad shape");
    const uintptr_t all = (uintptr_t)c->k_codes | (uintptr_t)c->v_codes | (uintptr_t)c->k_tail | (uintptr_t)c->v_tail;
    if (items && (!lengths || !c->k_tail || !c->v_tail || (c->table_width && !c->page_table) ||
                  (c->pages && (!c->k_codes || !c->v_codes || !c->k_scales || !c->v_scales)) || (all & 15)))
        return db_fail(DB_ERR_INVALID_ARGUMENT, "INVALID_ARGUMENT", name + ": missing or unaligned cache tensor");
    a->c = *c;
    a->lengths = lengths;
    a->cu = cu;
    a->items = (int)items;
    a->rows = (int)rows;
    a->max_rows = (int)max_rows;
    a->error = db_device_error_ptr();
    return DB_OK;
}

bool rows_ok(const void* p, int64_t ld, int64_t width) { return p && !((uintptr_t)p & 15) && !(ld & 7) && ld >= width; }

}  // namespace
}  // namespace db

extern "C" {

int db_kv8_append(const db_kv8_cache* cache, const void* k, int64_t ldk, const void* v, int64_t ldv,
                  const int32_t* lengths, const int32_t* cu_seqlens, int64_t items, int64_t rows, int64_t max_rows,
                  void* stream) {
    db::Kv8Args a{};
    const int rc = db::cache_args(cache, lengths, cu_seqlens, items, rows, max_rows, "kv8 append", &a);
    if (rc) return rc;
    if (items == 0 || max_rows == 0) return DB_OK;
    const int64_t width = (int64_t)cache->kv_heads * db::D;
    if (!db::rows_ok(k, ldk, width) || !db::rows_ok(v, ldv, width))
        return db_fail(DB_ERR_INVALID_ARGUMENT, "INVALID_ARGUMENT", "kv8 append: rows start on 16-byte boundaries");
    // blocks that max_rows tokens reach from the least favourable position
    const dim3 grid((unsigned)((db::BLK - 1 + max_rows - 1) / db::BLK + 1), cache->kv_heads, (unsigned)items);
    const dim3 block(db::APPEND_THREADS);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e =
        cache->dtype == DB_DTYPE_F16
            ? db_launch_pdl(db::kv8_append_kernel<__half>, grid, block, 0, s, a, static_cast<const __half*>(k), ldk,
                            static_cast<const __half*>(v), ldv)
            : db_launch_pdl(db::kv8_append_kernel<__nv_bfloat16>, grid, block, 0, s, a,
                            static_cast<const __nv_bfloat16*>(k), ldk, static_cast<const __nv_bfloat16*>(v), ldv);
    return db_cuda_status((int)e, "kv8 append");
}

int db_kv8_read(const db_kv8_cache* cache, const int32_t* lengths, int64_t items, int64_t max_keys, float* k, float* v,
                void* stream) {
    db::Kv8Args a{};
    const int rc = db::cache_args(cache, lengths, nullptr, items, 0, 0, "kv8 read", &a);
    if (rc) return rc;
    if (max_keys < 0 || max_keys >= ((int64_t)1 << 31) - db::BLK || (items && max_keys && (!k || !v || (((uintptr_t)k | (uintptr_t)v) & 15))))
        return db_fail(DB_ERR_INVALID_ARGUMENT, "INVALID_ARGUMENT", "kv8 read: bad shape");
    if (items == 0 || max_keys == 0) return DB_OK;
    const dim3 grid((unsigned)((max_keys + db::BLK - 1) / db::BLK * 2), cache->kv_heads, (unsigned)items);
    const dim3 block(db::READ_THREADS);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = cache->dtype == DB_DTYPE_F16
                              ? db_launch_pdl(db::kv8_read_kernel<__half>, grid, block, 0, s, a, max_keys, k, v)
                              : db_launch_pdl(db::kv8_read_kernel<__nv_bfloat16>, grid, block, 0, s, a, max_keys, k, v);
    return db_cuda_status((int)e, "kv8 read");
}

size_t db_kv8_attention_workspace_bytes(int64_t items, int64_t max_rows, int64_t max_keys, int64_t kv_heads,
                                        int64_t q_heads) {
    if (items <= 0 || max_rows <= 0 || max_keys <= 0 || kv_heads <= 0 || q_heads <= 0) return 0;
    const int nt = db::decode_tiles(max_rows * (q_heads / kv_heads));
    if (!nt) return 0;
    return (size_t)db::decode_ctas(items, kv_heads, max_keys) * db::DECODE_WARPS * 2 * db::part_floats(nt) * sizeof(float);
}

int db_kv8_attention(const db_kv8_cache* cache, const void* q, int64_t ldq, const int32_t* lengths,
                     const int32_t* cu_seqlens, int64_t items, int64_t rows, int64_t max_rows, int64_t max_keys,
                     int64_t q_heads, float scale, void* out, int64_t ldo, void* workspace, void* stream) {
    db::AttnArgs a{};
    const int rc = db::cache_args(cache, lengths, cu_seqlens, items, rows, max_rows, "kv8 attention", &a.kv);
    if (rc) return rc;
    if (q_heads <= 0 || q_heads % cache->kv_heads || q_heads > 65535 || max_keys <= 0)
        return db_fail(DB_ERR_INVALID_ARGUMENT, "INVALID_ARGUMENT", "kv8 attention: bad shape");
    if (items == 0 || max_rows == 0) return DB_OK;
    if (!db::rows_ok(q, ldq, q_heads * db::D) || !db::rows_ok(out, ldo, q_heads * db::D))
        return db_fail(DB_ERR_INVALID_ARGUMENT, "INVALID_ARGUMENT", "kv8 attention: rows start on 16-byte boundaries");
    a.q = q, a.ldq = ldq, a.out = out, a.ldo = ldo;
    a.group = (int)(q_heads / cache->kv_heads);
    a.factor = scale * 1.4426950408889634f;
    if ((int64_t)max_rows * a.group >= ((int64_t)1 << 31))
        return db_fail(DB_ERR_INVALID_ARGUMENT, "INVALID_ARGUMENT", "kv8 attention: bad shape");
    if (!workspace && db_kv8_attention_workspace_bytes(items, max_rows, max_keys, cache->kv_heads, q_heads))
        return db_fail(DB_ERR_INVALID_ARGUMENT, "INVALID_ARGUMENT", "kv8 attention: a workspace is needed");
    a.parts = static_cast<float*>(workspace);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = cache->dtype == DB_DTYPE_F16 ? db::attention<__half>(a, max_keys, s)
                                                       : db::attention<__nv_bfloat16>(a, max_keys, s);
    return db_cuda_status((int)e, "kv8 attention");
}

}  // extern "C"
