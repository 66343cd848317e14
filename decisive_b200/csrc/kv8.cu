// The 8-bit paged key/value cache (db_kv8_append, db_kv8_read) and the attention that reads it
// (db_kv8_attention).
//
// A sequence's tokens lie in blocks of 64.  A full block is one page of int8 codes per kv head with
// one f32 scale for its keys and one for its values: scale = max(max|x| * (1 / 127), FLT_MIN), code =
// round-half-even(x / scale).  The block that is still open is kept in 16 bits (the tail) and is
// quantised once, when its last token comes, so the codes do not depend on how the tokens were
// split over appends.  Keys are stored [64 tokens, 128], values [128, 64 tokens]: both are then
// read along the axis that their product sums over, 16 bytes at a time and without a transpose.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <float.h>

#include <type_traits>

#include "../../include/decisive_b200.h"
#include "capi_internal.h"
#include "common.cuh"
#include "kernels.h"

namespace cg = cooperative_groups;

namespace db {
namespace {

constexpr int D = 128, BLK = DB_KV8_BLOCK;

struct Kv8Args {
    db_kv8_cache c;
    const int32_t* lengths;  // [items] tokens cached before this call's rows
    const int32_t* cu;       // [items + 1] rows of the items, or null: max_rows each
    int items, rows, max_rows;
    int* error;
};

// Item b: rows [start, start + count) of this call, `len` tokens cached before them.  Offsets and
// lengths outside the tensors are brought back inside and noted in the error word.
__device__ __forceinline__ void item_of(const Kv8Args& a, int b, int& start, int& count, int& len) {
    if (a.cu) {
        start = min(max(a.cu[b], 0), a.rows);
        count = min(min(max(a.cu[b + 1], start), a.rows) - start, a.max_rows);
    } else {
        start = b * a.max_rows;
        count = a.max_rows;
    }
    const int64_t most = (int64_t)a.c.table_width * BLK;
    const int given = a.lengths[b];
    len = given;
    if (given < 0 || (int64_t)given + count > most) {
        len = given < 0 ? 0 : (int)min((int64_t)given, most);
        count = (int)min((int64_t)count, most - len);
        if (a.error && threadIdx.x == 0) atomicOr(a.error, DB_DEV_ERR_SHAPE);
    }
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
__device__ __forceinline__ void from_f32(float x, __half& y) { y = __float2half_rn(x); }
__device__ __forceinline__ void from_f32(float x, __nv_bfloat16& y) { y = __float2bfloat16_rn(x); }
template <typename T>
__device__ __forceinline__ float from_bits(uint32_t b) {
    const unsigned short h = (unsigned short)b;
    return to_f32(*reinterpret_cast<const T*>(&h));
}

// ------------------------------------------------------------------ append
constexpr int APPEND_THREADS = 256;
constexpr int V_PITCH = D + 2;  // elements: rows of the value tile start on different banks

// One CTA per touched block, kv head and item.  Its 64 x 128 keys and values are gathered from the
// tail and the new rows; a full block is quantised into its page, an open one keeps its new rows in
// the tail.  The first block's CTA also writes the tail of the last block, because the two use the
// same slots and it is the one that still reads them.  HBM bound; for one token it is launch
// latency, and only a block that fills up does more than copy 512 bytes.
template <typename T>
__global__ void __launch_bounds__(APPEND_THREADS)
    kv8_append_kernel(Kv8Args a, const T* __restrict__ k, int64_t ldk, const T* __restrict__ v, int64_t ldv) {
    __shared__ uint32_t largest[2];
    __shared__ __align__(16) T vt[BLK * V_PITCH];
    pdl_wait();
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
        for (int i = tid; i < n * D; i += APPEND_THREADS) {
            const int r = i / D, c = i % D, p = p0 + r;
            v_tail[c * BLK + p % BLK] = vrow[(int64_t)(p - len) * ldv + c];
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
    for (int e = tid; e < D * kept; e += APPEND_THREADS) {
        const int c = e / kept, r = e % kept;
        const T x = v_tail[c * BLK + r];
        vmax = max(vmax, (uint32_t) * reinterpret_cast<const unsigned short*>(&x) & 0x7fffu);
        vt[r * V_PITCH + c] = x;
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
        auto code = [](float x, float s) {
            const float c = rintf(__fdiv_rn(x, s));
            return (uint32_t)(c == c ? (int)fminf(fmaxf(c, -127.f), 127.f) : 0) & 0xffu;
        };
        int8_t* kp = a.c.k_codes + ph * BLK * D;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = tid + i * APPEND_THREADS;
            const uint32_t w[4] = {key[i].x, key[i].y, key[i].z, key[i].w};
            uint32_t o[2] = {0, 0};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                o[j >> 1] |= code(from_bits<T>(w[j] & 0xffffu), ks) << (16 * (j & 1));
                o[j >> 1] |= code(from_bits<T>(w[j] >> 16), ks) << (16 * (j & 1) + 8);
            }
            *reinterpret_cast<uint2*>(kp + (int64_t)e * 8) = make_uint2(o[0], o[1]);
        }
        int8_t* vp = a.c.v_codes + ph * D * BLK;
        for (int e = tid; e < D * BLK / 16; e += APPEND_THREADS) {
            const int c = e % D, r0 = e / D * 16;  // value feature c, tokens r0 .. r0 + 15
            uint32_t o[4] = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 16; ++j) o[j >> 2] |= code(to_f32(vt[(r0 + j) * V_PITCH + c]), vs) << (8 * (j & 3));
            *reinterpret_cast<uint4*>(vp + c * BLK + r0) = make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
    const int last = total / BLK;  // the block that stays open
    if (blockIdx.x == 0 && last > first && total % BLK) keep(last);
}

// ------------------------------------------------------------------ read back
// The cached values of tokens 0 .. max_keys - 1 in f32 (0 past an item's length).
template <typename T>
__global__ void kv8_read_kernel(Kv8Args a, int64_t max_keys, float* __restrict__ k, float* __restrict__ v) {
    __shared__ float tile[BLK][D + 1];
    const int tid = threadIdx.x, block = blockIdx.x, h = blockIdx.y, b = blockIdx.z, Hk = a.c.kv_heads;
    int start, count, len;
    item_of(a, b, start, count, len);
    const int n = (int)min((int64_t)BLK, max_keys - (int64_t)block * BLK);
    const bool full = (int64_t)(block + 1) * BLK <= len;
    const int inside = min(max(len - block * BLK, 0), BLK);
    const int page = full ? page_of(a, b, block) : -1;
    const int64_t ph = (int64_t)page * Hk + h, tail = ((int64_t)b * Hk + h) * BLK * D;
    for (int which = 0; which < 2; ++which) {
        const float scale = page >= 0 ? (which ? a.c.v_scales : a.c.k_scales)[ph] : 0.f;
        for (int e = tid; e < BLK * D; e += blockDim.x) {
            const int r = which ? e % BLK : e / D, c = which ? e / BLK : e % D;
            float x = 0.f;
            if (page >= 0)
                x = __fmul_rn((float)(which ? a.c.v_codes : a.c.k_codes)[ph * BLK * D + e], scale);
            else if (!full && r < inside)
                x = to_f32(static_cast<const T*>(which ? a.c.v_tail : a.c.k_tail)[tail + e]);
            tile[r][c] = x;
        }
        __syncthreads();
        float* out = (which ? v : k) + (((int64_t)b * max_keys + (int64_t)block * BLK) * Hk + h) * D;
        for (int e = tid; e < n * D; e += blockDim.x) out[(int64_t)(e / D) * Hk * D + e % D] = tile[e / D][e % D];
        __syncthreads();
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
// Four int8 codes as two pairs of f16, exactly: the bytes become the low bits of 1024 + (code + 128).
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
};

// Scores and the context are formed transposed, S^T = K Q^T and O^T = V^T P^T, so that the codes are
// the wide operand (16 keys or 16 value features of an MMA) and 8 query rows the narrow one: a single
// token's 4 or 8 heads fill it.  Row n of a kv head's tile is query (token n / group, head n % group).
//
// Every lane reads 16 codes in one load and they are exactly what its MMA fragments need, because
// the order of a product's sum is free: within a 64-wide half of a key, k step s of the fragment takes
// bytes 4s..4s+3 of each lane's 16; and key 16 (r >> 1) + 4 s + 2 half + (r & 1) sits in row r of
// half `half` of score tile s, which makes P^T's fragment the four bytes 4s..4s+3 of each 16 of V^T.
// Codes become f16 exactly; q is scaled by a power of two per row into f16 (bf16 has fewer bits
// and more range), so the scores' product rounds neither operand.  P is rounded after its f32 sum is
// taken, to one f16 for bf16 outputs and to two for f16 ones.  A block's own context is scaled by its value scale when
// it joins the running one, in f32.
//
// A warp takes whole blocks, with running maxima and sums of its own; the warps of a CTA and the
// CTAs of a cluster share a tile's keys and join once at the end, in a fixed order.
template <typename T, int NT>
struct Warp {
    float O[8][NT][4];
    float m[NT][2], l[NT][2];
};

template <typename T, int NT, int WARPS>
__global__ void __launch_bounds__(32 * WARPS) kv8_attention_kernel(AttnArgs a) {
    constexpr int ROWS = 8 * NT;
    constexpr bool TWO = std::is_same<T, __half>::value;
    extern __shared__ __align__(16) uint8_t attn_smem[];
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int split = cluster.block_rank(), splits = cluster.num_blocks();
    const int h = blockIdx.y, b = blockIdx.z, tile = blockIdx.x / splits, Hk = a.kv.c.kv_heads;
    // shared memory: query fragments and factors, then (over them) the joined results
    uint2* qfrag = reinterpret_cast<uint2*>(attn_smem);                // [NT][8][32]
    float* qfactor = reinterpret_cast<float*>(qfrag + NT * 8 * 32);    // [ROWS]
    pdl_wait();
    pdl_trigger();
    int start, count, len;
    item_of(a.kv, b, start, count, len);
    const int rows = count * a.group, row0 = tile * ROWS;
    if (row0 >= rows) return;  // the whole cluster leaves: tile is the cluster's
    const T* q = static_cast<const T*>(a.q);
    auto q_at = [&](int r) { return q + (int64_t)(start + r / a.group) * a.ldq + ((int64_t)h * a.group + r % a.group) * D; };

    // queries: one warp per row, 4 values a lane; scaled to [0.5, 1) x 2^8 at the row's largest value
    for (int r = warp; r < ROWS; r += WARPS) {
        float x[4] = {0.f, 0.f, 0.f, 0.f};
        if (row0 + r < rows) {
            const uint2 w = *reinterpret_cast<const uint2*>(q_at(row0 + r) + 4 * lane);
            x[0] = from_bits<T>(w.x & 0xffffu), x[1] = from_bits<T>(w.x >> 16);
            x[2] = from_bits<T>(w.y & 0xffffu), x[3] = from_bits<T>(w.y >> 16);
        }
        float top = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const int e = top > 0.f && top < INFINITY ? min(max(8 - ilogbf(top), -126), 126) : 0;
        const float up = ldexpf(1.f, e);
        if (lane == 0) qfactor[r] = ldexpf(1.f, -e);
        // dims 4 lane .. 4 lane + 3 = half c, quarter t' of it (16 dims), k step s
        const int c = lane >> 4, tt = (lane >> 2) & 3, s = lane & 3;
        qfrag[((r >> 3) * 8 + c * 4 + s) * 32 + (r & 7) * 4 + tt] =
            make_uint2(pack2<__half>(x[0] * up, x[1] * up), pack2<__half>(x[2] * up, x[3] * up));
    }
    __syncthreads();

    Warp<T, NT> w;
    float factor[NT][2];
    int limit[NT][2];  // last key that a column's row sees; -1: none
    int first_limit = 0x7fffffff, last_limit = -1;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int r = row0 + n * 8 + 2 * t + j;
            factor[n][j] = a.factor * qfactor[n * 8 + 2 * t + j];
            limit[n][j] = r < rows ? len + r / a.group : -1;
            w.m[n][j] = -INFINITY;
            w.l[n][j] = 0.f;
        }
    first_limit = len + row0 / a.group;
    last_limit = len + (min(row0 + ROWS, rows) - 1) / a.group;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) w.O[i][n][j] = 0.f;

    // S^T of one block is in s (16 keys per tile): softmax step; leaves P in f32 in s, returns the
    // factors of the running context
    auto soften = [&](float (&s)[4][NT][4], const float (&f)[NT][2], int base, float (&alpha)[NT][2]) {
        const bool masked = base + BLK - 1 > first_limit || row0 + ROWS > rows;
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
                const float now = fmaxf(w.m[n][j], top[j]);
                const float at = now == -INFINITY ? 0.f : now;
                alpha[n][j] = exp2f(w.m[n][j] - at);
                w.m[n][j] = now;
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const float p = exp2f(s[i][n][2 * half + j] - at);
                        s[i][n][2 * half + j] = p;
                        sum += p;
                    }
                w.l[n][j] = w.l[n][j] * alpha[n][j] + sum;
            }
        }
    };

    // this warp's blocks: the split's share, every WARPS-th
    const int blocks = last_limit / BLK + 1, whole = (len + count) / BLK;
    const int share = (blocks + splits - 1) / splits, from = split * share, to = min(from + share, blocks);
    for (int i = from + warp; i < to; i += WARPS) {
        if (i < whole) {
            const int page = page_of(a.kv, b, i);
            if (page < 0) continue;
            const int64_t ph = (int64_t)page * Hk + h;
            const int8_t* kp = a.kv.c.k_codes + ph * BLK * D;
            const int8_t* vp = a.kv.c.v_codes + ph * BLK * D;
            const float ks = a.kv.c.k_scales[ph], vs = a.kv.c.v_scales[ph];
            uint4 kc[4][2][2];  // score tile, row half, 64-wide half of the key
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int r = 0; r < 2; ++r)
#pragma unroll
                    for (int c = 0; c < 2; ++c)
                        kc[s][r][c] = __ldcs(reinterpret_cast<const uint4*>(
                            kp + (16 * (g >> 1) + 4 * s + 2 * r + (g & 1)) * D + 64 * c + 16 * t));
            float s[4][NT][4];
#pragma unroll
            for (int i2 = 0; i2 < 4; ++i2) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[i2][n][j] = 0.f;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const uint32_t lo[4] = {kc[i2][0][c].x, kc[i2][0][c].y, kc[i2][0][c].z, kc[i2][0][c].w};
                    const uint32_t hi[4] = {kc[i2][1][c].x, kc[i2][1][c].y, kc[i2][1][c].z, kc[i2][1][c].w};
#pragma unroll
                    for (int st = 0; st < 4; ++st) {
                        uint32_t f[4];
                        codes_to_f16(lo[st], f[0], f[2]);
                        codes_to_f16(hi[st], f[1], f[3]);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            const uint2 qf = qfrag[(n * 8 + c * 4 + st) * 32 + lane];
                            mma16(s[i2][n], f, qf.x, qf.y, __half());
                        }
                    }
                }
            }
            float alpha[NT][2], scaled[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 2; ++j) scaled[n][j] = factor[n][j] * ks;
            soften(s, scaled, i * BLK, alpha);
            // f16 outputs need P's next 11 bits as well: one rounding of P to f16 is as large as the output's
            uint32_t p[NT][4][2], rest[TWO ? NT : 1][4][2];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i2 = 0; i2 < 4; ++i2)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const float x = s[i2][n][2 * half], y = s[i2][n][2 * half + 1];
                        const uint32_t hi = pack2<__half>(x, y);
                        p[n][i2][half] = transpose8(hi);
                        if constexpr (TWO)
                            rest[n][i2][half] = transpose8(
                                pack2<__half>(x - from_bits<__half>(hi & 0xffffu), y - from_bits<__half>(hi >> 16)));
                    }
            float vf[NT][2];  // a block that a row does not see at all must not reach it (0 x NaN)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 2; ++j) vf[n][j] = limit[n][j] >= i * BLK ? vs : 0.f;
#pragma unroll
            for (int d = 0; d < 8; ++d) {
                const uint4 v0 = __ldcs(reinterpret_cast<const uint4*>(vp + (16 * d + g) * BLK + 16 * t));
                const uint4 v1 = __ldcs(reinterpret_cast<const uint4*>(vp + (16 * d + 8 + g) * BLK + 16 * t));
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
                        if constexpr (TWO) mma16(o[n], f, rest[n][st][0], rest[n][st][1], __half());
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        w.O[d][n][j] = fmaf(o[n][j], vf[n][j & 1], w.O[d][n][j] * alpha[n][j & 1]);
            }
        } else {
            // the open block, in 16 bits: the same walk on its own type
            const T* kt = static_cast<const T*>(a.kv.c.k_tail) + ((int64_t)b * Hk + h) * BLK * D;
            const T* vt = static_cast<const T*>(a.kv.c.v_tail) + ((int64_t)b * Hk + h) * BLK * D;
            const int inside = len + count - i * BLK;  // tokens of the block that are there
            float s[4][NT][4];
#pragma unroll
            for (int i2 = 0; i2 < 4; ++i2)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[i2][n][j] = 0.f;
#pragma unroll 1
            for (int c = 0; c < 2; ++c) {
                uint32_t qr[NT][8];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const int r = min(row0 + n * 8 + g, rows - 1);
                    const uint4* src = reinterpret_cast<const uint4*>(q_at(r) + 64 * c + 16 * t);
                    const uint4 x = src[0], y = src[1];
                    qr[n][0] = x.x, qr[n][1] = x.y, qr[n][2] = x.z, qr[n][3] = x.w;
                    qr[n][4] = y.x, qr[n][5] = y.y, qr[n][6] = y.z, qr[n][7] = y.w;
                }
#pragma unroll
                for (int i2 = 0; i2 < 4; ++i2) {
                    const int key = 16 * (g >> 1) + 4 * i2 + (g & 1);
                    const uint4* k0 = reinterpret_cast<const uint4*>(kt + key * D + 64 * c + 16 * t);
                    const uint4* k1 = reinterpret_cast<const uint4*>(kt + (key + 2) * D + 64 * c + 16 * t);
                    const uint4 a0 = k0[0], a1 = k0[1], b0 = k1[0], b1 = k1[1];
                    const uint32_t lo[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
                    const uint32_t hi[8] = {b0.x, b0.y, b0.z, b0.w, b1.x, b1.y, b1.z, b1.w};
#pragma unroll
                    for (int st = 0; st < 4; ++st) {
                        const uint32_t f[4] = {lo[2 * st], hi[2 * st], lo[2 * st + 1], hi[2 * st + 1]};
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma16(s[i2][n], f, qr[n][2 * st], qr[n][2 * st + 1], T());
                    }
                }
            }
            float alpha[NT][2], plain[NT][2];  // the queries come unscaled here
#pragma unroll
            for (int n = 0; n < NT; ++n) plain[n][0] = plain[n][1] = a.factor;
            soften(s, plain, i * BLK, alpha);
            // P in two parts of the tail's type, so that bf16 loses no more than f16
            uint32_t p[NT][4][2], rest[NT][4][2];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i2 = 0; i2 < 4; ++i2)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const float x = s[i2][n][2 * half], y = s[i2][n][2 * half + 1];
                        const uint32_t hi = pack2<T>(x, y);
                        const uint32_t lo = pack2<T>(x - from_bits<T>(hi & 0xffffu), y - from_bits<T>(hi >> 16));
                        p[n][i2][half] = transpose8(hi);
                        rest[n][i2][half] = transpose8(lo);
                    }
#pragma unroll
            for (int d = 0; d < 8; ++d) {
                float o[NT][4] = {};
                uint32_t f[2][8];
                bool odd = false;  // a NaN or an infinity among the values
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const uint4* src = reinterpret_cast<const uint4*>(vt + (16 * d + 8 * r + g) * BLK + 16 * t);
                    const uint4 x = src[0], y = src[1];
                    f[r][0] = x.x, f[r][1] = x.y, f[r][2] = x.z, f[r][3] = x.w;
                    f[r][4] = y.x, f[r][5] = y.y, f[r][6] = y.z, f[r][7] = y.w;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        // slots that hold no token yet, and what is not finite, stay out of the product
                        const int key = 16 * t + 2 * e;
                        uint32_t lo = f[r][e] & 0xffffu, hi = f[r][e] >> 16;
                        if (key >= inside) lo = 0;
                        if (key + 1 >= inside) hi = 0;
                        const bool bl = !isfinite(from_bits<T>(lo)), bh = !isfinite(from_bits<T>(hi));
                        odd |= bl | bh;
                        f[r][e] = (bl ? 0 : lo) | (bh ? 0 : hi) << 16;
                    }
                }
#pragma unroll
                for (int st = 0; st < 4; ++st) {
                    const uint32_t fa[4] = {f[0][2 * st], f[1][2 * st], f[0][2 * st + 1], f[1][2 * st + 1]};
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        mma16(o[n], fa, p[n][st][0], p[n][st][1], T());
                        mma16(o[n], fa, rest[n][st][0], rest[n][st][1], T());
                    }
                }
                if (__any_sync(0xffffffffu, odd)) {
                    // such a value reaches the rows that see its key, and no other
#pragma unroll
                    for (int r = 0; r < 2; ++r)
                        for (int key = 0; key < min(inside, BLK); ++key) {
                            const float x = to_f32(vt[(16 * d + 8 * r + g) * BLK + key]);
                            if (isfinite(x)) continue;
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int j = 0; j < 2; ++j)
                                    if (i * BLK + key <= limit[n][j]) o[n][2 * r + j] += x;
                        }
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int j = 0; j < 4; ++j) w.O[d][n][j] = fmaf(w.O[d][n][j], alpha[n][j & 1], o[n][j]);
            }
        }
    }

    // join: sums over the lanes that share a column, then the warps, then the cluster's CTAs
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int o = 4; o < 32; o *= 2) w.l[n][j] += __shfl_xor_sync(0xffffffffu, w.l[n][j], o);
    float* part_o = reinterpret_cast<float*>(attn_smem);          // [WARPS][ROWS][D + 4]
    float* part_m = part_o + WARPS * ROWS * (D + 4);              // [WARPS][ROWS]
    float* part_l = part_m + WARPS * ROWS;
    float* cta_m = part_l + WARPS * ROWS;                         // [ROWS]
    float* cta_l = cta_m + ROWS;
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int r = n * 8 + 2 * t + (j & 1);
#pragma unroll
            for (int d = 0; d < 8; ++d)
                part_o[(warp * ROWS + r) * (D + 4) + 16 * d + 8 * (j >> 1) + g] = w.O[d][n][j];
            if (g == 0 && j < 2) {
                part_m[warp * ROWS + r] = w.m[n][j];
                part_l[warp * ROWS + r] = w.l[n][j];
            }
        }
    __syncthreads();
    for (int e = tid; e < ROWS * D; e += 32 * WARPS) {
        const int r = e / D, c = e % D;
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < WARPS; ++i) m = fmaxf(m, part_m[i * ROWS + r]);
        const float at = m == -INFINITY ? 0.f : m;
        float o = 0.f, l = 0.f;
#pragma unroll
        for (int i = 0; i < WARPS; ++i) {
            const float f = exp2f(part_m[i * ROWS + r] - at);
            o = fmaf(part_o[(i * ROWS + r) * (D + 4) + c], f, o);
            l = fmaf(part_l[i * ROWS + r], f, l);
        }
        part_o[r * (D + 4) + c] = o;  // (this thread alone reads column c of row r)
        if (c == 0) cta_m[r] = m, cta_l[r] = l;
    }
    cluster.sync();
    for (int e = split * 32 * WARPS + tid; e < ROWS * D; e += splits * 32 * WARPS) {
        const int r = e / D, c = e % D, row = row0 + r;
        if (row >= rows) continue;
        float m = -INFINITY;
        for (int i = 0; i < splits; ++i) m = fmaxf(m, cluster.map_shared_rank(cta_m, i)[r]);
        const float at = m == -INFINITY ? 0.f : m;
        float o = 0.f, l = 0.f;
        for (int i = 0; i < splits; ++i) {
            const float f = exp2f(cluster.map_shared_rank(cta_m, i)[r] - at);
            o = fmaf(cluster.map_shared_rank(part_o, i)[r * (D + 4) + c], f, o);
            l = fmaf(cluster.map_shared_rank(cta_l, i)[r], f, l);
        }
        T y;
        from_f32(l == 0.f ? 0.f : o / l, y);  // l = 0: no key could be read
        static_cast<T*>(a.out)[(int64_t)(start + row / a.group) * a.ldo + ((int64_t)h * a.group + row % a.group) * D + c] = y;
    }
    cluster.sync();
}

template <typename T, int NT, int WARPS>
cudaError_t launch_attention(const AttnArgs& a, int tiles, int splits, cudaStream_t stream) {
    constexpr int ROWS = 8 * NT;
    constexpr int JOIN = WARPS * ROWS * (D + 4) * 4 + 2 * WARPS * ROWS * 4 + 2 * ROWS * 4;
    constexpr int FRAG = NT * 8 * 32 * 8 + ROWS * 4;
    constexpr int SMEM = JOIN > FRAG ? JOIN : FRAG;
    auto kernel = kv8_attention_kernel<T, NT, WARPS>;
    static thread_local int ready = -1;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (ready != dev) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
        ready = dev;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(tiles * splits, a.kv.c.kv_heads, a.kv.items);
    cfg.blockDim = dim3(32 * WARPS);
    cfg.dynamicSmemBytes = SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {(unsigned)splits, 1, 1};
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <typename T>
cudaError_t attention(const AttnArgs& a, int64_t max_keys, cudaStream_t stream) {
    const int64_t rows = (int64_t)a.kv.max_rows * a.group;
    const int nt = rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
    const int64_t tiles = (rows + 8 * nt - 1) / (8 * nt);
    const int64_t work = tiles * a.kv.c.kv_heads * a.kv.items, blocks = (max_keys + BLK - 1) / BLK;
    // split a tile's keys while that still finds idle SMs and every warp keeps a block
    int splits = 1;
    while (splits < 16 && work * splits < 2 * db_num_sms() && blocks > splits * 4) splits *= 2;
    if (tiles * splits > 0x7fffffff) return cudaErrorInvalidConfiguration;
    if (nt == 1) return launch_attention<T, 1, 4>(a, (int)tiles, splits, stream);
    if (nt == 2) return launch_attention<T, 2, 4>(a, (int)tiles, splits, stream);
    return launch_attention<T, 4, 4>(a, (int)tiles, splits, stream);
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
    if (max_keys < 0 || max_keys >= ((int64_t)1 << 31) - db::BLK || (items && max_keys && (!k || !v)))
        return db_fail(DB_ERR_INVALID_ARGUMENT, "INVALID_ARGUMENT", "kv8 read: bad shape");
    if (items == 0 || max_keys == 0) return DB_OK;
    const dim3 grid((unsigned)((max_keys + db::BLK - 1) / db::BLK), cache->kv_heads, (unsigned)items);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (cache->dtype == DB_DTYPE_F16)
        db::kv8_read_kernel<__half><<<grid, 256, 0, s>>>(a, max_keys, k, v);
    else
        db::kv8_read_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(a, max_keys, k, v);
    return db_cuda_status((int)cudaGetLastError(), "kv8 read");
}

int db_kv8_attention(const db_kv8_cache* cache, const void* q, int64_t ldq, const int32_t* lengths,
                     const int32_t* cu_seqlens, int64_t items, int64_t rows, int64_t max_rows, int64_t max_keys,
                     int64_t q_heads, float scale, void* out, int64_t ldo, void* stream) {
    db::AttnArgs a{};
    const int rc = db::cache_args(cache, lengths, cu_seqlens, items, rows, max_rows, "kv8 attention", &a.kv);
    if (rc) return rc;
    if (q_heads <= 0 || q_heads % cache->kv_heads || q_heads > 65535 || max_keys < 0)
        return db_fail(DB_ERR_INVALID_ARGUMENT, "INVALID_ARGUMENT", "kv8 attention: bad shape");
    if (items == 0 || max_rows == 0) return DB_OK;
    if (!db::rows_ok(q, ldq, q_heads * db::D) || !db::rows_ok(out, ldo, q_heads * db::D))
        return db_fail(DB_ERR_INVALID_ARGUMENT, "INVALID_ARGUMENT", "kv8 attention: rows start on 16-byte boundaries");
    a.q = q, a.ldq = ldq, a.out = out, a.ldo = ldo;
    a.group = (int)(q_heads / cache->kv_heads);
    a.factor = scale * 1.4426950408889634f;
    if ((int64_t)max_rows * a.group >= ((int64_t)1 << 31))
        return db_fail(DB_ERR_INVALID_ARGUMENT, "INVALID_ARGUMENT", "kv8 attention: bad shape");
    const int64_t most = (int64_t)cache->table_width * db::BLK;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = cache->dtype == DB_DTYPE_F16 ? db::attention<__half>(a, max_keys ? max_keys : most, s)
                                                       : db::attention<__nv_bfloat16>(a, max_keys ? max_keys : most, s);
    return db_cuda_status((int)e, "kv8 attention");
}

}  // extern "C"
