// The gated delta rule (db_gated_delta): per sequence and value head a state S [128 value, 128 key]
// in f32 and, token by token,
//   S <- e^g S;  u = beta (v - S k);  S <- S + u k^T;  o = S q
// with k and q divided by their lengths (norm_eps >= 0) and q times `scale`.
#include <cuda_bf16.h>

#include <type_traits>

#include "../../include/decisive_b200.h"
#include "capi_internal.h"
#include "common.cuh"
#include "kernels.h"
#include "tc_chain.cuh"

namespace db {
namespace {

constexpr int D = 128;  // head width: the state is D x D

struct DeltaArgs {
    const void *q, *k, *v;
    int64_t ldq, ldk, ldv;  // row strides, elements
    const float *g, *beta;
    int64_t ldg, ldb;
    const int32_t* cu;  // [items + 1], or null: items of max_len rows
    int items, rows, max_len, k_heads, v_heads;
    float scale, eps;
    const float* state_in;  // null: zeros
    int64_t state_stride;   // floats between the items' initial states (0: one for all)
    float* state_out;       // null: not kept
    void* out;
    int64_t ldo;
};

// Item b's rows [start, end); offsets outside the tensors are brought back inside them.
__device__ __forceinline__ void item_rows(const DeltaArgs& a, int b, int& start, int& end) {
    if (a.cu) {
        start = min(max(a.cu[b], 0), a.rows);
        end = min(max(a.cu[b + 1], start), a.rows);
    } else {
        start = b * a.max_len;
        end = start + a.max_len;
    }
}

template <typename T>
__device__ __forceinline__ float4 load4(const T* p);
template <>
__device__ __forceinline__ float4 load4<__half>(const __half* p) {
    const uint2 r = *reinterpret_cast<const uint2*>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&r.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&r.y));
    return make_float4(a.x, a.y, b.x, b.y);
}
template <>
__device__ __forceinline__ float4 load4<__nv_bfloat16>(const __nv_bfloat16* p) {
    const uint2 r = *reinterpret_cast<const uint2*>(p);
    return make_float4(__uint_as_float(r.x << 16), __uint_as_float(r.x & 0xffff0000u), __uint_as_float(r.y << 16),
                       __uint_as_float(r.y & 0xffff0000u));
}
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_f32(float x, __half& y) { y = __float2half_rn(x); }
__device__ __forceinline__ void from_f32(float x, __nv_bfloat16& y) { y = __float2bfloat16_rn(x); }

__device__ __forceinline__ float dot4(float4 a, float4 b) {
    return fmaf(a.w, b.w, fmaf(a.z, b.z, fmaf(a.y, b.y, a.x * b.x)));
}
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

// The recurrence as it is written, for items of few tokens (above all one): HBM bound, 64 KB of
// state read and written per item and head.  A warp owns 8 value rows of one state (lane l the keys
// 4l..4l+3, so each row is one 512-byte access) and never meets another warp.  Both products of a
// token are taken from the old state, S_new q = e^g S q + u (k.q), so the rows' 16 sums fold
// together: 16 values over 32 lanes in 16 shuffles, after which lane l holds sum l / 2.
// B200, 128 items of one token, 32 heads: 80 us, 6.7 TB/s, the copy's rate; one item: 15 us, launch latency.
constexpr int STEP_ROWS = 8, STEP_WARPS = 4;

template <typename T>
__global__ void __launch_bounds__(32 * STEP_WARPS) delta_step_kernel(DeltaArgs a) {
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row0 = (blockIdx.x * STEP_WARPS + warp) * STEP_ROWS;  // value rows row0 .. row0 + 7
    const int hv = blockIdx.y, b = blockIdx.z;
    const int hk = (int)((int64_t)hv * a.k_heads / a.v_heads);
    int start, end;
    item_rows(a, b, start, end);

    float4 S[STEP_ROWS];
    const int64_t at = ((int64_t)hv * D + row0) * D + 4 * lane;
    if (a.state_in) {
        const float* s = a.state_in + (int64_t)b * a.state_stride + at;
#pragma unroll
        for (int i = 0; i < STEP_ROWS; ++i) S[i] = *reinterpret_cast<const float4*>(s + i * D);
    } else {
#pragma unroll
        for (int i = 0; i < STEP_ROWS; ++i) S[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const T* q = static_cast<const T*>(a.q) + (int64_t)hk * D + 4 * lane;
    const T* k = static_cast<const T*>(a.k) + (int64_t)hk * D + 4 * lane;
    const int mine = (lane >> 1) & 7;  // the value row whose sums end in this lane
    const T* v = static_cast<const T*>(a.v) + (int64_t)hv * D + row0 + mine;
    T* out = static_cast<T*>(a.out) + (int64_t)hv * D + row0 + mine;
    for (int64_t t = start; t < end; ++t) {
        const float4 kk = load4(k + t * a.ldk), qq = load4(q + t * a.ldq);
        const float vv = to_f32(v[t * a.ldv]);
        const float decay = expf(a.g[t * a.ldg + hv]), beta = a.beta[t * a.ldb + hv];
        float kn = 1.f, qn = a.scale;
        if (a.eps >= 0.f) {
            kn = rsqrtf(warp_sum(dot4(kk, kk)) + a.eps);
            qn = rsqrtf(warp_sum(dot4(qq, qq)) + a.eps) * a.scale;
        }
        const float kq = warp_sum(dot4(kk, qq)) * kn * qn;
        // sums 0..7: S k of the rows, 8..15: S q
        float x[16];
#pragma unroll
        for (int i = 0; i < STEP_ROWS; ++i) {
            x[i] = dot4(S[i], kk);
            x[8 + i] = dot4(S[i], qq);
        }
#pragma unroll
        for (int w = 8; w; w >>= 1) {
            const bool up = lane & (2 * w);
#pragma unroll
            for (int i = 0; i < w; ++i) {
                const float give = up ? x[i] : x[i + w], keep = up ? x[i + w] : x[i];
                x[i] = keep + __shfl_xor_sync(0xffffffffu, give, 2 * w);
            }
        }
        x[0] += __shfl_xor_sync(0xffffffffu, x[0], 1);
        // lanes 0..15 hold S k of row lane / 2, lanes 16..31 S q of row (lane - 16) / 2
        const float sq = __shfl_down_sync(0xffffffffu, x[0], 16);
        const float u = beta * (vv - decay * kn * x[0]);  // (lanes 0..15)
        if (lane < 16 && !(lane & 1)) from_f32(fmaf(u, kq, decay * qn * sq), out[t * a.ldo]);
        const float uk = u * kn;
#pragma unroll
        for (int i = 0; i < STEP_ROWS; ++i) {
            const float w = __shfl_sync(0xffffffffu, uk, 2 * i);
            S[i].x = fmaf(w, kk.x, decay * S[i].x);
            S[i].y = fmaf(w, kk.y, decay * S[i].y);
            S[i].z = fmaf(w, kk.z, decay * S[i].z);
            S[i].w = fmaf(w, kk.w, decay * S[i].w);
        }
    }
    if (a.state_out) {
        float* s = a.state_out + (int64_t)b * a.v_heads * D * D + at;
#pragma unroll
        for (int i = 0; i < STEP_ROWS; ++i) *reinterpret_cast<float4*>(s + i * D) = S[i];
    }
}

// ------------------------------------------------------------------ chunks of 64 tokens
// With G_i the sum of g over a chunk's tokens up to i, K and Q the normalised rows and S0 the state before
// the chunk,
//   A_ij = beta_i e^(G_i - G_j) k_i.k_j (j < i),  T = (I + A)^-1 diag(beta),  P_ij = e^(G_i - G_j) q_i.k_j (j <= i)
//   U = T (V - diag(e^G) K S0^T),  O = diag(e^G) Q S0^T + P U,  S1 = e^G_C S0 + sum_i e^(G_C - G_i) u_i k_i^T
// (the chunked form of the delta rule that was published as "Parallelizing Linear Transformers with the Delta Rule over
// Sequence Length", 2024, with decays).  T and P need no state: delta_prepare_kernel forms them for all chunks at once;
// delta_chain_kernel then walks a sequence's chunks.  Chunks of 64: the walk's steps are a chain whose length is the number
// of chunks, and 64 is the largest chunk whose triangles' parts fit in shared memory twice.  B200, 16 key and 32 value
// heads: 512 tokens 55 us, 8229 tokens 629 us (48 TFLOP/s counted as the recurrence), 64 items of 16 to 1024 tokens 1.00 ms
// (124 TFLOP/s).
//
// Numerics.  The state has to keep f32's accuracy through f16 tensor products: k and q enter them exactly (as f16 after a
// power of two per row, which loses nothing within 2^-24 of the row's largest value; f16 queries as they are; their lengths
// are applied afterwards as factors per token.  Keys need the power in f16 too: the factors of U' hold 1 / |k|, and one short
// key would push the other tokens' U' into f16's subnormals), and every f32 operand (S, R, U, T, P) as the sum of two f16
// parts after a power of two: per row of the state for S and R, per chunk for T and P, so that 22 bits remain of what
// matters: a token whose values lie 2^-20 below the largest of their feature in its chunk keeps fewer, a row of the state
// likewise under terms that its own decay has since removed.  lo x lo products are left out (2^-22).  Decay sums are taken in
// f64: differences of f32 sums would lose what a slow decay has left.
constexpr int C = 64;                    // tokens per chunk
constexpr int BLOCKS = 10;               // 16 x 16 blocks of a lower triangle of 64, 512 bytes each, row-major
constexpr int TRI = BLOCKS * 256;        // halves of one triangle
// floats per chunk and head: factors per token of R (times S k), O (times S q) and U' (times U), then numbers of the chunk
enum Factor { F_R = 0, F_O = C, F_U = 2 * C, F_DECAY = 3 * C, F_T, F_P, F_OMEGA, F_REACH, F_GROW, FACTORS = 3 * C + 8 };

struct ChunkSpace {
    __half *k16, *q16;  // the rows as f16 after their powers, [chunk ids][C][k_heads][D]; q16: null for f16 inputs
    __half* tri;        // [chunk ids][v_heads][4][TRI]: T hi, T lo, P hi, P lo
    float* factor;      // [chunk ids][v_heads][FACTORS]
};

// Chunk ids: item b's chunks start at start_b / C + b, which leaves every item room for all of its chunks.
__host__ __device__ inline int64_t chunk_ids(int64_t rows, int64_t items) { return rows / C + items; }

size_t chunk_space(int64_t items, int64_t rows, int k_heads, int v_heads, bool queries, uint8_t* base, ChunkSpace* w) {
    const int64_t n = chunk_ids(rows, items);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        uint8_t* p = base ? base + at : nullptr;
        at += (bytes + 255) / 256 * 256;
        return p;
    };
    ChunkSpace s{};
    s.k16 = reinterpret_cast<__half*>(take((size_t)n * C * k_heads * D * 2));
    if (queries) s.q16 = reinterpret_cast<__half*>(take((size_t)n * C * k_heads * D * 2));
    s.tri = reinterpret_cast<__half*>(take((size_t)n * v_heads * 4 * TRI * 2));
    s.factor = reinterpret_cast<float*>(take((size_t)n * v_heads * FACTORS * 4));
    if (w) *w = s;
    return at;
}

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
// Byte offset of 16-byte piece c of row r in a tile of 256-byte rows (pieces permuted per row so that eight
// rows of one column of pieces lie on different banks).
__device__ __forceinline__ uint32_t tile_at(int r, int c) { return (uint32_t)(r * 256 + ((c ^ (r & 7)) << 4)); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <typename T>
__device__ __forceinline__ float lane16(uint32_t bits) {
    const unsigned short u = (unsigned short)bits;
    return to_f32(*reinterpret_cast<const T*>(&u));
}

// 2^e that brings a largest magnitude m into [2^14, 2^15) (1 for 0, infinities and NaN), and 2^-e.
__device__ __forceinline__ float row_power(float m, float& back) {
    const int e = (int)((__float_as_uint(m) >> 23) & 0xff) - 127;
    const int k = m > 0.f && e < 128 ? min(max(14 - e, -126), 126) : 0;
    back = __uint_as_float((uint32_t)(127 - k) << 23);
    return __uint_as_float((uint32_t)(127 + k) << 23);
}
// x, y as f16 pairs hi + lo
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}

constexpr int PREP_THREADS = 128;
constexpr int AP = 68;  // row pitch of the f32 triangles, floats (rows stay 16-byte aligned)

struct PrepShared {
    union {
        struct {
            uint8_t k[C * 256], q[C * 256];  // f16 tiles
        };
        struct {
            float A[C * AP], T[C * AP];      // once the products are in registers
        };
    };
    float tmp[32 * 36];
    float Gh[PREP_THREADS / 32][C], Gl[PREP_THREADS / 32][C];  // per head of a batch: decay sums (log2) in two parts: their differences keep what one would round away
    float beta[PREP_THREADS / 32][C], rk[C], rq[C], nk[C];
    float top[2][PREP_THREADS / 32];
};

__device__ __forceinline__ float2 pair_of(const float* x, int at) { return *reinterpret_cast<const float2*>(x + at); }

// o[i] = sum over k < depth of a[i][k] b[k], rows of a AP apart, b's entries ldb: two products to an instruction.
template <int R, int STEP>
__device__ __forceinline__ void block_product(float (&o)[R], const float* a, const float* b, int ldb, int depth) {
    uint64_t sum[R];
#pragma unroll
    for (int i = 0; i < R; ++i) sum[i] = 0;
#pragma unroll 1
    for (int k0 = 0; k0 < depth; k0 += STEP)
#pragma unroll
        for (int k = k0; k < k0 + STEP; k += 4) {
            const uint64_t y0 = f2_pack(__float_as_uint(b[k * ldb]), __float_as_uint(b[(k + 1) * ldb]));
            const uint64_t y1 = f2_pack(__float_as_uint(b[(k + 2) * ldb]), __float_as_uint(b[(k + 3) * ldb]));
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(a + i * AP + k);
                sum[i] = f2_fma(x.y, y1, f2_fma(x.x, y0, sum[i]));
            }
        }
#pragma unroll
    for (int i = 0; i < R; ++i) o[i] = f2_lo(sum[i]) + f2_hi(sum[i]);
}

// T, P and the factors of one chunk, for one key head and `heads` of the value heads that share it.  K K^T and Q K^T on
// mma.sync, once for the value heads of a key head; the inverse by blocks, -T11 A10 T00 from 16 x 16 to 64 x 64, in f32, because
// an f16 product would lose what the state is to keep.  Bound by shared memory's latency
// and wavefronts (58% of their rate; issue 47%) and the barriers between its short steps, which 4 CTAs an SM cover in part.
// B200: 0.40 ms of the 1.00 ms of 64 items, 0.10 ms of the 0.63 of 8229 tokens.
template <typename T>
__global__ void __launch_bounds__(PREP_THREADS, 4) delta_prepare_kernel(DeltaArgs a, ChunkSpace w, int heads) {
    extern __shared__ __align__(16) uint8_t prep_smem[];
    PrepShared& sh = *reinterpret_cast<PrepShared*>(prep_smem);
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int id = blockIdx.x, hk = blockIdx.y;
    // the item whose chunk this is: the last one that starts at or before id
    int lo = 0, hi = a.items - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        int s, e;
        item_rows(a, mid, s, e);
        if (s / C + mid <= id) lo = mid; else hi = mid - 1;
    }
    int start, end;
    item_rows(a, lo, start, end);
    const int row0 = start + (id - (start / C + lo)) * C;
    if (row0 < start || row0 >= end) return;
    const int n = min(C, end - row0);

    // warp i of a batch of heads forms the factors of its i-th head; its gates are loaded ahead of the tiles
    constexpr int WARPS = PREP_THREADS / 32;
    const int group = a.v_heads / a.k_heads, first = hk * group + blockIdx.z * heads, last = min(first + heads, (hk + 1) * group);
    float gate[2] = {}, beta[2] = {};
    auto load_gates = [&](int batch) {
        if (batch + warp >= last) return;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int i = 2 * lane + j;
            gate[j] = i < n ? a.g[(int64_t)(row0 + i) * a.ldg + batch + warp] : 0.f;
            beta[j] = i < n ? a.beta[(int64_t)(row0 + i) * a.ldb + batch + warp] : 0.f;
        }
    };
    auto factors = [&](int batch) {
        if (batch + warp >= last) return;
        float* factor = w.factor + ((int64_t)id * a.v_heads + batch + warp) * FACTORS;
        double x[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            x[j] = gate[j] < -1e4f ? -1e4 : (double)gate[j];  // e^-10000 = 0; -inf would make differences NaN
            sh.beta[warp][2 * lane + j] = beta[j];
        }
        double sum = x[0] + x[1];
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const double y = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += y;
        }
        const double all = __shfl_sync(0xffffffffu, sum, 31);
        float fu[2], reach = 0.f, largest = 0.f, grow = 0.f;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int i = 2 * lane + j;
            const double G = j ? sum : sum - x[1], two = G * 1.4426950408889634;
            sh.Gh[warp][i] = (float)two;
            sh.Gl[warp][i] = (float)(two - (double)sh.Gh[warp][i]);
            const float e = expf((float)G);
            factor[F_R + i] = e * sh.rk[i];
            factor[F_O + i] = e * sh.rq[i];
            const float left = expf((float)(all - G));
            fu[j] = left * sh.rk[i];
            grow += left * sh.nk[i];
            reach = fmaxf(reach, e * sh.nk[i]);
            largest = fmaxf(largest, fabsf(fu[j]));
        }
        reach = warp_max(reach);
        largest = warp_max(largest);
        grow = warp_sum(grow);
        float back;
        const float omega = row_power(largest, back) * (1.f / 65536.f);  // factors of U' to at most 1/2
        factor[F_U + 2 * lane] = fu[0] * omega;
        factor[F_U + 2 * lane + 1] = fu[1] * omega;
        if (lane == 0) {
            factor[F_DECAY] = expf((float)all);
            factor[F_OMEGA] = back * 65536.f;
            factor[F_REACH] = 11.4f * reach;  // |S k| <= sqrt(128) |k| max |S|
            factor[F_GROW] = omega * grow;    // |sum U'_i k_i| <= max |U| sum of the weights
        }
    };
    load_gates(first);

    // rows into shared memory as f16, with their factors
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const bool scaled = which == 0 || !std::is_same<T, __half>::value;
        const T* src = static_cast<const T*>(which ? a.q : a.k) + (int64_t)hk * D;
        const int64_t ld = which ? a.ldq : a.ldk;
        uint4 raw[8];
#pragma unroll
        for (int it = 0; it < 8; ++it) {
            const int r = warp * 16 + it * 2 + (lane >> 4), c = lane & 15;
            raw[it] = r < n ? *reinterpret_cast<const uint4*>(src + (int64_t)(row0 + r) * ld + 8 * c) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int it = 0; it < 8; ++it) {
            const int r = warp * 16 + it * 2 + (lane >> 4), c = lane & 15;
            float x[8];
            const T* p = reinterpret_cast<const T*>(&raw[it]);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = to_f32(p[j]);
            float ss = 0.f, top = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                ss = fmaf(x[j], x[j], ss);
                top = fmaxf(top, fabsf(x[j]));
            }
#pragma unroll
            for (int o = 8; o; o >>= 1) {
                ss += __shfl_xor_sync(0xffffffffu, ss, o);
                if (scaled) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            }
            float back = 1.f;
            uint4 y = raw[it];
            if (scaled) {
                // 2^6 below the other operands' scale: products of two rows stay far inside f32
                const float up = row_power(top, back) * 0.015625f;
                back *= 64.f;
                uint32_t o4[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const __half2 h = __floats2half2_rn(x[2 * j] * up, x[2 * j + 1] * up);
                    o4[j] = *reinterpret_cast<const uint32_t*>(&h);
                }
                y = make_uint4(o4[0], o4[1], o4[2], o4[3]);
                __half* dst = (which ? w.q16 : w.k16) + (((int64_t)id * C + r) * a.k_heads + hk) * D + 8 * c;
                *reinterpret_cast<uint4*>(dst) = y;
            }
            *reinterpret_cast<uint4*>((which ? sh.q : sh.k) + tile_at(r, c)) = y;
            if (c == 0) {
                // (a row of zeros, past the end or given, takes no part: its 1 / sqrt(eps) must not set the others' scale)
                const float inverse = ss == 0.f ? 0.f : a.eps >= 0.f ? rsqrtf(ss + a.eps) : 1.f;
                (which ? sh.rq : sh.rk)[r] = inverse * (which ? a.scale : 1.f) * back;
                if (!which) sh.nk[r] = sqrtf(ss) * inverse;
            }
        }
    }
    __syncthreads();

    factors(first);
    // K K^T and Q K^T, rows 16 warp .. + 15, columns up to the diagonal
    float kk[8][4], qk[8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) kk[j][i] = qk[j][i] = 0.f;
    const uint32_t sk = smem_u32(sh.k), sq = smem_u32(sh.q);
#pragma unroll
    for (int s = 0; s < 8; ++s) {
        uint32_t ak[4], aq[4];
        const uint32_t off = tile_at(warp * 16 + (lane & 15), 2 * s + (lane >> 4));
        ldmatrix4(ak, sk + off);
        ldmatrix4(aq, sq + off);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j <= warp) {
                uint32_t b[4];  // two n tiles: rows 16 j .. + 15 of K
                ldmatrix4(b, sk + tile_at(16 * j + ((lane >> 4) << 3) + (lane & 7), 2 * s + ((lane >> 3) & 1)));
                mma16816(kk[2 * j], ak, b[0], b[1]);
                mma16816(kk[2 * j + 1], ak, b[2], b[3]);
                mma16816(qk[2 * j], aq, b[0], b[1]);
                mma16816(qk[2 * j + 1], aq, b[2], b[3]);
            }
    }

    for (int hv = first; hv < last; ++hv) {
        const int h = (hv - first) % WARPS;
        if (h == 0) {
            if (hv > first) {
                __syncthreads();
                load_gates(hv);
                factors(hv);
            }
            __syncthreads();  // the tiles, or the last head's triangles, have been read; the factors are there
        }
        __half* tri = w.tri + ((int64_t)id * a.v_heads + hv) * 4 * TRI;
        float* factor = w.factor + ((int64_t)id * a.v_heads + hv) * FACTORS;
        const float *Ghs = sh.Gh[h], *Gls = sh.Gl[h], *betas = sh.beta[h];
        // A into shared memory, P to its place
        float p[8][4], largest = 0.f, row_Gh[2], row_Gl[2], row_k[2], row_q[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = warp * 16 + g + 8 * i;
            row_Gh[i] = Ghs[r], row_Gl[i] = Gls[r], row_k[i] = sh.rk[r] * betas[r], row_q[i] = sh.rq[r];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < 2 * warp + 2) {
                const int c0 = 8 * j + 2 * t;
                const float2 Gh = pair_of(Ghs, c0), Gl = pair_of(Gls, c0), rk = pair_of(sh.rk, c0);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int r = warp * 16 + g + 8 * i;
                    const float d0 = c0 <= r ? ex2((row_Gh[i] - Gh.x) + (row_Gl[i] - Gl.x)) * rk.x : 0.f;
                    const float d1 = c0 + 1 <= r ? ex2((row_Gh[i] - Gh.y) + (row_Gl[i] - Gl.y)) * rk.y : 0.f;
                    float* x = &p[j][2 * i];
                    *reinterpret_cast<float2*>(&sh.A[r * AP + c0]) = make_float2(c0 < r ? kk[j][2 * i] * d0 * row_k[i] : 0.f,
                                                                                 c0 + 1 < r ? kk[j][2 * i + 1] * d1 * row_k[i] : 0.f);
                    x[0] = c0 <= r ? qk[j][2 * i] * d0 * row_q[i] : 0.f;
                    x[1] = c0 + 1 <= r ? qk[j][2 * i + 1] * d1 * row_q[i] : 0.f;
                    largest = fmaxf(largest, fmaxf(fabsf(x[0]), fabsf(x[1])));
                }
            }
        largest = warp_max(largest);
        if (lane == 0) sh.top[0][warp] = largest;
        // two f16 parts after one power of two for the whole triangle; rows of 16 x 16 blocks
        auto store = [&](float (&x)[8][4], const float (&top)[PREP_THREADS / 32], int which, int f) {
            float back;
            const float up = row_power(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), back);
            if (tid == 0) factor[f] = back;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j < 2 * warp + 2)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        uint32_t h, l;
                        split2(x[j][2 * i] * up, x[j][2 * i + 1] * up, h, l);
                        const int at = (warp * (warp + 1) / 2 + (j >> 1)) * 256 + (g + 8 * i) * 16 + 8 * (j & 1) + 2 * t;
                        *reinterpret_cast<uint32_t*>(tri + which * TRI + at) = h;
                        *reinterpret_cast<uint32_t*>(tri + (which + 1) * TRI + at) = l;
                    }
        };
        __syncthreads();
        store(p, sh.top[0], 2, F_P);
        // (I + A)^-1, 16 x 16 blocks on the diagonal: lane c < 16 of warp b solves for column c of block b
        if (lane < 16) {
            const float* Ab = sh.A + (16 * warp) * AP + 16 * warp;
            float x[16];  // each entry, once it is known, leaves all later ones: the sums do not wait for one another
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = i == lane ? 1.f : 0.f;
#pragma unroll
            for (int j = 0; j < 15; j += 4)
#pragma unroll
                for (int i = j + 1; i < 16; ++i) {  // (A's entries from the diagonal on are zero)
                    const float4 y = *reinterpret_cast<const float4*>(Ab + i * AP + j);
                    x[i] = fmaf(-y.x, x[j], x[i]);
                    if (j + 1 < i) x[i] = fmaf(-y.y, x[j + 1], x[i]);
                    if (j + 2 < i) x[i] = fmaf(-y.z, x[j + 2], x[i]);
                    if (j + 3 < i) x[i] = fmaf(-y.w, x[j + 3], x[i]);
                }
#pragma unroll
            for (int i = 0; i < 16; ++i) sh.T[(16 * warp + i) * AP + 16 * warp + lane] = x[i];
        }
        __syncthreads();
        // the block below two neighbours: -T11 A10 T00, first for 16 x 16 blocks, then for 32 x 32
        {
            const int pr = tid >> 6, c = tid & 15, r0 = ((tid >> 4) & 3) * 4, b0 = 32 * pr;
            float o[4];
            block_product<4, 16>(o, sh.A + (b0 + 16 + r0) * AP + b0, sh.T + b0 * AP + b0 + c, AP, 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) sh.tmp[(16 * pr + r0 + i) * 36 + c] = o[i];
            __syncthreads();
            float z[4];
            block_product<4, 16>(z, sh.T + (b0 + 16 + r0) * AP + b0 + 16, sh.tmp + 16 * pr * 36 + c, 36, 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) sh.T[(b0 + 16 + r0 + i) * AP + b0 + c] = -z[i];
            // the 16 x 16 blocks above the diagonal are zero
#pragma unroll
            for (int i = 0; i < 4; ++i) sh.T[(b0 + r0 + i) * AP + b0 + 16 + c] = 0.f;
        }
        __syncthreads();
        {
            const int c = lane, r0 = warp * 8;
            float o[8];
            block_product<8, 16>(o, sh.A + (32 + r0) * AP, sh.T + c, AP, 32);
#pragma unroll
            for (int i = 0; i < 8; ++i) sh.tmp[(r0 + i) * 36 + c] = o[i];
            __syncthreads();
            float z[8];  // (T11's rows end at the diagonal)
            block_product<8, 8>(z, sh.T + (32 + r0) * AP + 32, sh.tmp + c, 36, r0 + 8);
#pragma unroll
            for (int i = 0; i < 8; ++i) sh.T[(32 + r0 + i) * AP + c] = -z[i];
        }
        __syncthreads();
        largest = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < 2 * warp + 2) {
                const int c0 = 8 * j + 2 * t;
                const float2 beta = pair_of(betas, c0);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int r = warp * 16 + g + 8 * i;
                    const float2 y = pair_of(sh.T, r * AP + c0);
                    float* x = &p[j][2 * i];
                    x[0] = c0 <= r ? y.x * beta.x : 0.f;
                    x[1] = c0 + 1 <= r ? y.y * beta.y : 0.f;
                    largest = fmaxf(largest, fmaxf(fabsf(x[0]), fabsf(x[1])));
                }
            }
        largest = warp_max(largest);
        if (lane == 0) sh.top[1][warp] = largest;
        __syncthreads();
        store(p, sh.top[1], 0, F_T);
    }
}

__device__ __forceinline__ void cp_async16_if(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

// Walks the chunks of one item and value head.  Latency bound: four products follow one another per chunk, each taking
// f16 parts of what the one before left, so the state's 128 value rows are the 128 lanes of tensor memory, every product
// has them as its rows (A from tensor memory, B from shared memory), and nothing of the chain passes through shared
// memory:
//   X = S [K; Q]^T,  R = V - e^G X_k,  U = R T^T,  S <- e^G_C S + U' K,  O = e^G X_q + U P^T
// The state stays in tensor memory as its two parts (22 bits and the second part's sign: off by 2^-23 of a value at most,
// where f32 would be by 2^-24; 129 chunks with hardly any decay stay within 6e-6 of its RMS); tensor-core sums enter it by
// one f32 fma, because the cores' own accumulation truncates.  The powers of two that keep parts in range come from bounds,
// max |S k| <= sqrt(128) |k| max |S| for R, e^G_C max |S| + max |U| sum e^(G_C-G_i) |k_i| for the next S; the slack of a
// bound (2^6) costs nothing, because f16 parts of a row scaled to 2^15 reach down to 2^-40 of it.
// The code is kept small: what the warps of an SM run between two products has to stay in its instruction cache.
// B200: 8000 cycles per chunk, most of them the rows' arithmetic and hand-offs (16 warps for the rows instead of 8 were
// no faster).  One CTA per SM (shared memory, all of tensor memory), so one item of 32 heads keeps 32 SMs busy.
//
// Warps 0-7: the rows' arithmetic (thread: row 32 (w & 3) + lane; tokens 32 (w >> 2) .. + 31, or these and the keys 64 further on);
// 8: MMA issue and tensor memory; 9-11: loads of the next chunk, outputs of the last.
// Tensor memory columns: S parts 0-127, U' K 128-255, U 256-319 (then U' parts in its place), P U 320-383, X_k 384-447
// (then R parts, then U parts), X_q 448-511.  Parts of 32 values lie in 32 columns: 16 of first parts (two values to a
// column), 16 of second parts.
constexpr int CHAIN_THREADS = 384, LOADERS = 96;
constexpr uint64_t DRAIN_NS = 100000000ull;
constexpr int KQ_BYTES = 2 * C * D * 2, KQ_HALF = KQ_BYTES / 2, TRI_BYTES = C * C * 2;

struct ChainStage {
    uint8_t kq[KQ_BYTES];       // rows 0-63 K, 64-127 Q; two columns of 64 keys x 128 rows, 128-byte swizzle
    uint8_t tri[4][TRI_BYTES];  // T hi, T lo, P hi, P lo: 64 rows of 128 bytes, 128-byte swizzle
    uint8_t v[C * D * 2];
};
enum ChainBar { CB_FULL = 0, CB_EMPTY = 2, CB_S = 4, CB_D = 6, CB_X = 8, CB_R, CB_U, CB_W, CB_UU, CB_PU, CB_OUT, CB_SENT, CB_DONE, CB_END, CHAIN_BARS };
struct ChainShared {
    uint8_t out[C * D * 2];  // a chunk's outputs on their way
    uint64_t bars[CHAIN_BARS];
    alignas(16) float factor[2][FACTORS];
    float top[3][2][D];  // largest magnitudes of S, U and V: [half][row]
    uint32_t tmem;
    int abort;
};
constexpr int CHAIN_SMEM = 1024 + 2 * sizeof(ChainStage) + sizeof(ChainShared);
static_assert(sizeof(ChainStage) % 1024 == 0 && CHAIN_SMEM <= 232448, "shared memory");

// B operand with N contiguous (MN-major), 128-byte swizzle: rows of 128 bytes hold 64 values of N for one K; 8-row atoms
// are 1024 bytes apart, the next 64 values of N KQ_HALF bytes.
__device__ __forceinline__ uint64_t mn_desc(uint32_t smem_addr) {
    return (uint64_t)((smem_addr >> 4) & 0x3FFFu) | (uint64_t)((KQ_HALF >> 4) & 0x3FFFu) << 16 |
           (uint64_t)(1024u >> 4) << 32 | (uint64_t)1u << 46 | (uint64_t)2u << 61;
}
// 32 values (16 pairs) as f16 parts: 16 columns of first parts, 16 of second ones.
__device__ __forceinline__ void parts32(const uint64_t (&x)[16], uint32_t (&r)[32]) {
    const uint64_t minus = f2_pack(0xbf800000u, 0xbf800000u);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const __half2 h = __floats2half2_rn(f2_lo(x[i]), f2_hi(x[i]));
        const float2 f = __half22float2(h);
        const uint64_t left = f2_fma(f2_pack(__float_as_uint(f.x), __float_as_uint(f.y)), minus, x[i]);
        const __half2 l = __floats2half2_rn(f2_lo(left), f2_hi(left));
        r[i] = *reinterpret_cast<const uint32_t*>(&h);
        r[16 + i] = *reinterpret_cast<const uint32_t*>(&l);
    }
}
__device__ __forceinline__ uint64_t both(float x) { return f2_pack(__float_as_uint(x), __float_as_uint(x)); }
// Four factors of neighbouring tokens from shared memory.
__device__ __forceinline__ ulonglong2 pairs_at(const float* f) { return *reinterpret_cast<const ulonglong2*>(f); }

template <typename T>
__global__ void __launch_bounds__(CHAIN_THREADS, 1) delta_chain_kernel(DeltaArgs a, ChunkSpace w, int* err) {
    extern __shared__ uint8_t chain_smem[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(chain_smem) + 1023) & ~uintptr_t(1023));
    ChainStage* stages = reinterpret_cast<ChainStage*>(smem);
    ChainShared& sh = *reinterpret_cast<ChainShared*>(smem + 2 * sizeof(ChainStage));
    volatile int* abort_flag = &sh.abort;
    const int tid = threadIdx.x, lane = tid & 31, warp = chain::warp_index();
    const int hv = blockIdx.x, b = blockIdx.y, hk = hv / (a.v_heads / a.k_heads);
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.bars[CB_FULL + i], LOADERS / 32);
            mbar_init(&sh.bars[CB_EMPTY + i], 1 + 8);
            mbar_init(&sh.bars[CB_S + i], 8);
            mbar_init(&sh.bars[CB_D + i], 1);
        }
        for (int i : {CB_R, CB_W, CB_UU, CB_OUT}) mbar_init(&sh.bars[i], 8);
        mbar_init(&sh.bars[CB_SENT], LOADERS / 32);
        for (int i : {CB_X, CB_U, CB_PU, CB_DONE}) mbar_init(&sh.bars[i], 1);
        mbar_init(&sh.bars[CB_END], CHAIN_THREADS / 32);
        sh.abort = 0;
        fence_barrier_init();
    }
    if (warp == 8) {
        tmem_alloc(&sh.tmem, 512);
        tmem_relinquish();
    }
    pdl_wait();
    pdl_trigger();
    int start, end;
    item_rows(a, b, start, end);
    const int chunks = (end - start + C - 1) / C;
    const int64_t id0 = start / C + b;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;

    if (warp >= 9) {
        // ---------------------------------------------------------------- loads
        const int lt = tid - 9 * 32;
        bool ok = true;
        // chunk c's outputs from shared memory, 16 bytes at a time
        auto send = [&](int c) {
            ok = ok && chain::warp_wait(&sh.bars[CB_OUT], c & 1, abort_flag, err, DB_DEV_ERR_TIMEOUT_EPI);
            if (!ok) return;
            const int row0 = start + c * C, n = min(C, end - row0);
            T* out = static_cast<T*>(a.out) + (int64_t)row0 * a.ldo + (int64_t)hv * D;
            for (int r = lt >> 4; r < n; r += LOADERS / 16)
                *reinterpret_cast<uint4*>(out + (int64_t)r * a.ldo + 8 * (lt & 15)) =
                    *reinterpret_cast<const uint4*>(sh.out + r * (D * 2) + 16 * (lt & 15));
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.bars[CB_SENT]);
        };
        for (int c = 0; c <= chunks && ok; ++c) {
            if (c > 0) {
                // the chunk before has landed: to the tensor core's view, then on
                cp_async_wait<0>();
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.bars[CB_FULL + ((c - 1) & 1)]);
            }
            if (c < chunks) {
                const int s = c & 1;
                ok = chain::warp_wait(&sh.bars[CB_EMPTY + s], ((c >> 1) & 1) ^ 1u, abort_flag, err, DB_DEV_ERR_TIMEOUT_TMA);
                if (!ok) break;
                ChainStage& st = stages[s];
                const int row0 = start + c * C, n = min(C, end - row0);
                const int64_t id = id0 + c;
                const __half* k16 = w.k16 + (id * C * a.k_heads + hk) * D;
                const __half* q16 = w.q16 ? w.q16 + (id * C * a.k_heads + hk) * D
                                          : static_cast<const __half*>(a.q) + (int64_t)row0 * a.ldq + (int64_t)hk * D;
                const int64_t ldk = (int64_t)a.k_heads * D, ldq = w.q16 ? (int64_t)a.k_heads * D : a.ldq;
                const uint32_t skq = smem_u32(st.kq), sv = smem_u32(st.v), stri = smem_u32(st.tri);
                // 16-byte piece p of row r: column p / 8, place p % 8 ^ r % 8
                const int p16 = lt & 15, r16 = lt >> 4;
                for (int r = r16; r < C; r += LOADERS / 16) {
                    const bool there = r < n;
                    const int rr = there ? r : 0;
                    const uint32_t to = skq + (p16 >> 3) * KQ_HALF + r * 128 + (((p16 & 7) ^ (r & 7)) << 4);
                    cp_async16_if(to, k16 + rr * ldk + 8 * p16, there);
                    cp_async16_if(to + C * 128, q16 + rr * ldq + 8 * p16, there);
                    cp_async16_if(sv + r * (D * 2) + 16 * p16,
                                  static_cast<const T*>(a.v) + (int64_t)(row0 + rr) * a.ldv + (int64_t)hv * D + 8 * p16, there);
                }
                // the triangles' blocks: 32 pieces each, row x of the block, half y
                const __half* tri = w.tri + (id * a.v_heads + hv) * 4 * TRI;
                const int x = lane >> 1, y = lane & 1;
                for (int e = warp - 9; e < 4 * BLOCKS; e += LOADERS / 32) {
                    const int which = e / BLOCKS, blk = e % BLOCKS;
                    const int I = blk >= 6 ? 3 : blk >= 3 ? 2 : blk >= 1 ? 1 : 0, J = blk - I * (I + 1) / 2;
                    cp_async16_if(stri + which * TRI_BYTES + (16 * I + x) * 128 + (((2 * J + y) ^ (x & 7)) << 4),
                                  tri + which * TRI + blk * 256 + x * 16 + y * 8, true);
                }
                const float* f = w.factor + (id * a.v_heads + hv) * FACTORS;
                for (int e = lt; e < FACTORS / 4; e += LOADERS) cp_async16_if(smem_u32(&sh.factor[s][4 * e]), f + 4 * e, true);
                cp_async_commit();
            }
            if (c > 1) send(c - 2);  // (formed at the start of chunk c - 1)
        }
        if (chunks > 0) send(chunks - 1);
        cp_async_wait<0>();
    } else if (warp == 8) {
        // ---------------------------------------------------------------- MMA issue
        // Six jobs a chunk, one loop body: X from the first and the last 64 keys, U, U' K for the first and the last 64
        // keys, P U.  (Halves, because the state's arithmetic before X and after U' K goes by halves too.)
        const uint32_t tmem = __shfl_sync(0xffffffffu, sh.tmem, 0);  // (uniform, for the compiler)
        bool ok = true;
        auto wait = [&](int bar, uint32_t parity) {
            ok = ok && chain::warp_wait(&sh.bars[bar], parity, abort_flag, err, DB_DEV_ERR_TIMEOUT_MMA);
            tc_fence_after();
        };
        for (int c = 0; c < chunks && ok; ++c) {
            const int s = c & 1;
            const uint32_t ph = c & 1;
            const uint32_t kq = smem_u32(stages[s].kq);
            const uint64_t dT = sw128_desc(smem_u32(stages[s].tri));
            if (c > 0) wait(CB_PU, ph ^ 1u);  // (X goes where its U parts were)
            wait(CB_FULL + s, (c >> 1) & 1);
#pragma unroll 1
            for (int job = 0; job < 6 && ok; ++job) {
                // a triangle's K step k meets rows 16 k .. of it only
                const bool tri = job == 2 || job == 5, state = job < 2;
                const uint32_t half = job & 1;  // (of X, job 0 and 1, and of U' K, jobs 3 and 4: 1 for the first half)
                wait(state ? CB_S + job : job == 2 ? CB_R : job == 5 ? CB_UU : CB_W, ph);
                const uint32_t d = tmem + (state ? 384u : job == 2 ? 256u : job == 5 ? 320u : 192u - 64u * half);
                const uint32_t a_tm = tmem + (state ? 64u * job : tri ? 384u : 256u);
                const uint64_t b0 = state ? sw128_desc(kq + KQ_HALF * job) : job == 2 ? dT : job == 5 ? dT + (2 * TRI_BYTES >> 4) : mn_desc(kq + KQ_HALF * (1u - half));
                const uint32_t id0 = state ? idesc_f16_f32(128, 128) : tri ? idesc_f16_f32(128, 64) : idesc_f16_f32(128, 64) | (1u << 16);
                const uint32_t b_step = state ? 2u : tri ? 130u : 128u;
                if (chain::elect()) {
#pragma unroll 1
                    for (uint32_t k = 0; k < 4; ++k) {
                        const uint32_t at = a_tm + 32u * (k >> 1) + 8u * (k & 1), dk = tri ? d + 16u * k : d;
                        const uint32_t id = tri ? id0 - k * (2u << 17) : id0;
                        const uint64_t b = b0 + (uint64_t)(k * b_step);
                        chain::umma_f16_ts(dk, at + 16u, b, id, k > 0 || job == 1);
                        if (tri) chain::umma_f16_ts(dk, at, b + (TRI_BYTES >> 4), id, 1);
                        chain::umma_f16_ts(dk, at, b, id, 1);
                    }
                    if (job > 0) umma_commit(&sh.bars[job == 1 ? CB_X : job == 2 ? CB_U : job == 5 ? CB_PU : CB_D + job - 3]);
                    if (job == 5) umma_commit(&sh.bars[CB_EMPTY + s]);
                }
                __syncwarp();
            }
        }
        // every MMA issued has completed before tensor memory is released
        if (chain::elect()) {
            umma_commit(&sh.bars[CB_DONE]);
            mbar_wait_drain(&sh.bars[CB_DONE], 0, DRAIN_NS);
        }
        __syncwarp();
    } else {
        // ---------------------------------------------------------------- the rows' arithmetic
        const int half = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t tm = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        bool ok = true;
        auto wait = [&](int bar, uint32_t parity) {
            ok = ok && chain::warp_wait(&sh.bars[bar], parity, abort_flag, err, DB_DEV_ERR_TIMEOUT_EPI);
            tc_fence_after();
            return ok;
        };
        auto ready = [&](int bar) {  // what this warp stored in tensor memory may be read
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.bars[bar]);
        };
        float s_top = 0.f;  // the row's largest S part (of these keys until the halves meet)
        // largest magnitude among first parts (rounding moves it by 2^-11, which the bounds below allow for)
        auto parts_top = [](const uint32_t (&r)[32], __half2 top) {
#pragma unroll
            for (int i = 0; i < 16; ++i) top = __hmax2(top, __habs2(*reinterpret_cast<const __half2*>(&r[i])));
            return top;
        };
        auto top_of = [](__half2 x) { return __half2float(__hmax(__low2half(x), __high2half(x))); };
        // a power of two 2^e (e of a float's exponent field) and the next one for a largest magnitude of `bound`
        int up_e = 0;  // S parts hold S 2^up_e
        auto power = [](int e) { return __uint_as_float((uint32_t)(127 + e) << 23); };
        auto retarget = [&](float bound) {  // the step that brings bound to [2^14, 2^15)
            const int e = (int)((__float_as_uint(bound) >> 23) & 0xff) - 127;
            const int step = bound > 0.f && e < 128 ? 14 - e : 0;
            return min(max(max(step, -100), -100 - up_e), min(100, 100 - up_e));
        };
        const int64_t at = ((int64_t)hv * D + row) * D + 32 * half;  // this thread's keys: 32 half .. + 31, and 64 further on
        if (chunks > 0) {
            // the state that is given, looked at once for its largest value, then split
            float top = 0.f;
            const float* in = a.state_in ? a.state_in + (int64_t)b * a.state_stride + at : nullptr;
            if (in)
#pragma unroll 4
                for (int i = 0; i < 16; ++i) {
                    const float4 x = *reinterpret_cast<const float4*>(in + 4 * i + 32 * (i >> 3));
                    top = fmaxf(fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))), top);
                }
            sh.top[0][half][row] = top;
            named_barrier_sync(1, 256);
            top = fmaxf(top, sh.top[0][half ^ 1][row]);
            up_e = retarget(top);
            s_top = top * power(up_e);
            named_barrier_sync(1, 256);
            const uint64_t up = both(power(up_e));
#pragma unroll 1
            for (int q = 0; q < 2; ++q) {
                uint64_t x[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = in ? f2_mul(*reinterpret_cast<const uint64_t*>(in + 64 * q + 2 * i), up) : 0ull;
                uint32_t r[32];
                parts32(x, r);
                chain::tmem_st32(tm + 64u * q + 32u * half, r);
                ready(CB_S + q);
            }
        }
        uint64_t Oq[16];
        float o_scale = 0.f;
        // chunk c's outputs: e^G S q is there, P U joins it; they leave through shared memory
        auto output = [&](int c) {
            if (c > 0) wait(CB_SENT, (c - 1) & 1);
            uint32_t r[32];
            tmem_ld_32x32b_x32(tm + 320u + 32u * half, r);
            tmem_wait_ld(r);
            T* out = reinterpret_cast<T*>(sh.out) + 32 * half * D + row;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const uint64_t o = f2_fma(f2_pack(r[2 * i], r[2 * i + 1]), both(o_scale), Oq[i]);
                from_f32(f2_lo(o), out[2 * i * D]);
                from_f32(f2_hi(o), out[(2 * i + 1) * D]);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.bars[CB_OUT]);
        };
        // (after an abort the waits return at once and the rest runs on: every warp meets the barriers as often as the others)
        for (int c = 0; c < chunks; ++c) {
            const int s = c & 1;
            const uint32_t ph = c & 1;
            const float* f = sh.factor[s];
            uint32_t r[32];
            uint64_t x[16];
            // while X is formed: V, and the chunk before goes out
            wait(CB_FULL + s, (c >> 1) & 1);
            uint32_t V[16], v_bits = 0;
            {
                const unsigned short* v = reinterpret_cast<const unsigned short*>(stages[s].v) + 32 * half * D + row;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    V[i] = (uint32_t)v[2 * i * D] | (uint32_t)v[(2 * i + 1) * D] << 16;
                    v_bits = __vmaxu2(v_bits, V[i] & 0x7fff7fffu);
                }
            }
            sh.top[0][half][row] = s_top;
            sh.top[2][half][row] = lane16<T>(max(v_bits & 0xffffu, v_bits >> 16));
            if (c > 0) {
                wait(CB_PU, ph ^ 1u);
                output(c - 1);
            }
            named_barrier_sync(1, 256);
            s_top = fmaxf(s_top, sh.top[0][half ^ 1][row]);
            const float v_top = fmaxf(sh.top[2][0][row], sh.top[2][1][row]);
            // R = V - e^G S k
            const float s_back = power(-up_e);
            float r_back;
            const float r_up = row_power(v_top + f[F_REACH] * (s_top * s_back), r_back);
            wait(CB_X, ph);
            tmem_ld_32x32b_x32(tm + 384u + 32u * half, r);
            tmem_wait_ld(r);
            {
                const uint64_t k = both(-s_back * r_up), up = both(r_up);
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    const ulonglong2 w = pairs_at(f + F_R + 32 * half + 2 * i);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint64_t vv = f2_pack(__float_as_uint(lane16<T>(V[i + j] & 0xffffu)), __float_as_uint(lane16<T>(V[i + j] >> 16)));
                        x[i + j] = f2_fma(f2_mul(f2_pack(r[2 * i + 2 * j], r[2 * i + 2 * j + 1]), k), j ? w.y : w.x, f2_mul(vv, up));
                    }
                }
                parts32(x, r);
            }
            chain::tmem_st32(tm + 384u + 32u * half, r);
            ready(CB_R);
            // while U is formed: e^G S q
            tmem_ld_32x32b_x32(tm + 448u + 32u * half, r);
            tmem_wait_ld(r);
            {
                const uint64_t k = both(s_back);
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    const ulonglong2 w = pairs_at(f + F_O + 32 * half + 2 * i);
                    Oq[i] = f2_mul(f2_mul(f2_pack(r[2 * i], r[2 * i + 1]), k), w.x);
                    Oq[i + 1] = f2_mul(f2_mul(f2_pack(r[2 * i + 2], r[2 * i + 3]), k), w.y);
                }
            }
            // U in units of 2^22 / (r_up x T's power): at most 2^14 whatever R and T are
            const float u_back = 4194304.f * r_back * f[F_T], grow = f[F_GROW];
            o_scale = u_back * f[F_P];
            const float s_scale = u_back * f[F_OMEGA] * power(up_e), decay = f[F_DECAY];
            wait(CB_U, ph);
            tmem_ld_32x32b_x32(tm + 256u + 32u * half, r);
            tmem_wait_ld(r);
            {
                const uint64_t k = both(2.3841858e-7f);
                uint64_t y[16];
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    const ulonglong2 w = pairs_at(f + F_U + 32 * half + 2 * i);
                    x[i] = f2_mul(f2_pack(r[2 * i], r[2 * i + 1]), k);
                    x[i + 1] = f2_mul(f2_pack(r[2 * i + 2], r[2 * i + 3]), k);
                    y[i] = f2_mul(x[i], w.x);
                    y[i + 1] = f2_mul(x[i + 1], w.y);
                }
                parts32(y, r);
            }
            chain::tmem_st32(tm + 256u + 32u * half, r);
            ready(CB_W);
            parts32(x, r);
            chain::tmem_st32(tm + 384u + 32u * half, r);
            ready(CB_UU);
            // while U' K is formed: what the next chunk's powers of two need
            const float u_top = top_of(parts_top(r, __half2{}));
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.bars[CB_EMPTY + s]);  // this warp is done with the chunk's values and factors
            sh.top[1][half][row] = u_top;
            named_barrier_sync(1, 256);
            const int step = retarget(decay * s_top + fmaxf(u_top, sh.top[1][half ^ 1][row]) * grow * fabsf(s_scale));
            up_e += step;
            const uint64_t keep = both(decay * power(step)), add = both(s_scale * power(step));
            // S <- e^G_C S + U' K
            __half2 top{};
#pragma unroll 1
            for (int q = 0; q < 2; ++q) {
                uint32_t d[32];
                wait(CB_D + q, ph);
                tmem_ld_32x32b_x32(tm + 64u * q + 32u * half, r);
                tmem_ld_32x32b_x32(tm + 128u + 64u * q + 32u * half, d);
                tmem_wait_ld(r);
                chain::tie32(d);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&r[i])), l = __half22float2(*reinterpret_cast<const __half2*>(&r[16 + i]));
                    const uint64_t old = f2_add(f2_pack(__float_as_uint(h.x), __float_as_uint(h.y)), f2_pack(__float_as_uint(l.x), __float_as_uint(l.y)));
                    x[i] = f2_fma(f2_pack(d[2 * i], d[2 * i + 1]), add, f2_mul(old, keep));
                }
                parts32(x, r);
                chain::tmem_st32(tm + 64u * q + 32u * half, r);
                ready(CB_S + q);  // (half of the next X is formed while the other half is updated)
                top = parts_top(r, top);
            }
            s_top = top_of(top);
        }
        if (chunks > 0) {
            wait(CB_PU, (chunks - 1) & 1);
            output(chunks - 1);
        }
        if (a.state_out && ok) {
            float* o = a.state_out + (int64_t)b * a.v_heads * D * D + at;
            const float back = power(-up_e);
#pragma unroll 1
            for (int q = 0; q < 2; ++q) {
                uint32_t r[32];
                if (chunks > 0) {
                    tmem_ld_32x32b_x32(tm + 64u * q + 32u * half, r);
                    tmem_wait_ld(r);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (chunks > 0) {
                        const float2 h0 = __half22float2(*reinterpret_cast<const __half2*>(&r[2 * i])), l0 = __half22float2(*reinterpret_cast<const __half2*>(&r[16 + 2 * i]));
                        const float2 h1 = __half22float2(*reinterpret_cast<const __half2*>(&r[2 * i + 1])), l1 = __half22float2(*reinterpret_cast<const __half2*>(&r[17 + 2 * i]));
                        y = make_float4((h0.x + l0.x) * back, (h0.y + l0.y) * back, (h1.x + l1.x) * back, (h1.y + l1.y) * back);
                    } else if (a.state_in) {
                        y = *reinterpret_cast<const float4*>(a.state_in + (int64_t)b * a.state_stride + at + 64 * q + 4 * i);
                    }
                    *reinterpret_cast<float4*>(o + 64 * q + 4 * i) = y;
                }
            }
        }
    }
    // through an mbarrier: every role is done with tensor memory before it is released
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.bars[CB_END]);
    if (warp == 8) {
        if (lane == 0) mbar_wait_drain(&sh.bars[CB_END], 0, DB_WAIT_LIMIT_NS);
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Up to this many tokens per item the recurrence runs, whatever the items: one number, because callers size the workspace by
// it.  It is on the safe side of both crossings (recurrence / chunks, us, 32 heads, 128 items: 8 tokens 216 / 564, 16 385 / 568,
// 24 559 / 575, 32 731 / 577; one item: 8 11 / 34, 16 14 / 34, 32 25 / 34, 48 33 / 34, 64 43 / 34).
constexpr int STEP_TOKENS = DB_DELTA_STEP_TOKENS;

template <typename T>
cudaError_t launch(const DeltaArgs& a, void* workspace, cudaStream_t stream) {
    if (a.max_len <= STEP_TOKENS) {
        const dim3 grid(D / (STEP_ROWS * STEP_WARPS), a.v_heads, a.items);
        return db_launch_pdl(delta_step_kernel<T>, grid, dim3(32 * STEP_WARPS), 0, stream, a);
    }
    ChunkSpace w;
    chunk_space(a.items, a.rows, a.k_heads, a.v_heads, !std::is_same<T, __half>::value, static_cast<uint8_t*>(workspace), &w);
    cudaError_t e = db_set_max_smem(reinterpret_cast<const void*>(delta_prepare_kernel<T>), sizeof(PrepShared));
    if (e != cudaSuccess) return e;
    // a CTA per value head while that still finds idle SMs, else one for all that share a key head (per value head / per
    // key head, us of the whole call: 512 tokens 58 / 62, 8229 tokens 664 / 632, 64 items of 16 to 1024 tokens 1144 / 1004)
    const int64_t ids = chunk_ids(a.rows, a.items);
    const int group = a.v_heads / a.k_heads, heads = ids * a.k_heads < 4 * db_num_sms() ? 1 : group;
    e = db_launch_pdl(delta_prepare_kernel<T>, dim3((unsigned)ids, a.k_heads, (group + heads - 1) / heads), dim3(PREP_THREADS),
                      sizeof(PrepShared), stream, a, w, heads);
    if (e != cudaSuccess) return e;
    e = db_set_max_smem(reinterpret_cast<const void*>(delta_chain_kernel<T>), CHAIN_SMEM);
    if (e != cudaSuccess) return e;
    return db_launch_pdl(delta_chain_kernel<T>, dim3(a.v_heads, a.items), dim3(CHAIN_THREADS), CHAIN_SMEM, stream, a, w,
                         db_device_error_ptr());
}

// Whether a final state lies over an initial state that is not its own item's: other CTAs would read what it writes.
// stride: floats between initial states, one: floats of a state.
bool states_meet(const float* in, int64_t stride, const float* out, int64_t items, int64_t one) {
    if (!in || !out || (in == out && (items == 1 || stride == one))) return false;
    // in floats from the first initial state: the final ones cover [begin, end); a wide stride leaves gaps between the initial
    const int64_t begin = ((intptr_t)out - (intptr_t)in) / (int64_t)sizeof(float), end = begin + items * one;
    if (stride == 0) return begin < one && end > 0;
    const int64_t first = begin < one ? 0 : (begin - one) / stride + 1;  // the first item whose state ends past begin
    return first < items && first * stride < end;
}

}  // namespace
}  // namespace db

extern "C" {

size_t db_gated_delta_workspace_bytes(int64_t items, int64_t rows, int64_t max_len, int64_t k_heads, int64_t v_heads,
                                      int dtype) {
    if (max_len <= db::STEP_TOKENS || items <= 0 || rows <= 0 || k_heads <= 0 || v_heads <= 0) return 0;
    return db::chunk_space(items, rows, (int)k_heads, (int)v_heads, dtype != DB_DTYPE_F16, nullptr, nullptr);
}

int db_gated_delta(const void* q, const void* k, const void* v, int dtype, int64_t ldq, int64_t ldk, int64_t ldv,
                   const float* g, const float* beta, int64_t ldg, int64_t ldb, const int32_t* cu_seqlens,
                   int64_t items, int64_t rows, int64_t max_len, int64_t k_heads, int64_t v_heads, int64_t head_dim,
                   float scale, float norm_eps, const float* state_in, int64_t state_stride, float* state_out,
                   void* out, int64_t ldo, void* workspace, void* stream) {
    if (head_dim != 128)
        return db_fail(DB_ERR_UNSUPPORTED, "UNSUPPORTED", "gated delta rule: head_dim must be 128");
    if (dtype != DB_DTYPE_F16 && dtype != DB_DTYPE_BF16)
        return db_fail(DB_ERR_UNSUPPORTED, "UNSUPPORTED", "gated delta rule: q, k and v are f16 or bf16");
    const int64_t most = (int64_t)1 << 31;
    if (items < 0 || rows < 0 || max_len < 0 || rows >= most || items > 65535 || k_heads <= 0 || v_heads <= 0 ||
        v_heads > 65535 || v_heads % k_heads || max_len > rows || (!cu_seqlens && rows != items * max_len))
        return db_fail(DB_ERR_INVALID_ARGUMENT, "INVALID_ARGUMENT", "gated delta rule: bad shape");
    if (items == 0) return DB_OK;
    if (rows > 0 && (!q || !k || !v || !g || !beta || !out || ldq < k_heads * 128 || ldk < k_heads * 128 ||
                     ldv < v_heads * 128 || ldo < v_heads * 128 || ldg < v_heads || ldb < v_heads))
        return db_fail(DB_ERR_INVALID_ARGUMENT, "INVALID_ARGUMENT", "gated delta rule: missing tensor or short row");
    const uintptr_t all = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)state_in |
                          (uintptr_t)state_out | (uintptr_t)workspace;
    if ((all & 15) || ((ldq | ldk | ldv | ldo) & 7) || (state_stride & 3))
        return db_fail(DB_ERR_INVALID_ARGUMENT, "INVALID_ARGUMENT",
                       "gated delta rule: rows and states start on 16-byte boundaries");
    if (state_in && state_stride != 0 && state_stride < v_heads * 128 * 128)
        return db_fail(DB_ERR_INVALID_ARGUMENT, "INVALID_ARGUMENT", "gated delta rule: states overlap");
    if (db::states_meet(state_in, state_stride, state_out, items, v_heads * 128 * 128))
        return db_fail(DB_ERR_INVALID_ARGUMENT, "INVALID_ARGUMENT",
                       "gated delta rule: a state can be updated in place only by its own item");
    if (!workspace && db_gated_delta_workspace_bytes(items, rows, max_len, k_heads, v_heads, dtype))
        return db_fail(DB_ERR_INVALID_ARGUMENT, "INVALID_ARGUMENT", "gated delta rule: a workspace is needed");
    db::DeltaArgs a{};
    a.q = q, a.k = k, a.v = v;
    a.ldq = ldq, a.ldk = ldk, a.ldv = ldv;
    a.g = g, a.beta = beta;
    a.ldg = ldg, a.ldb = ldb;
    a.cu = cu_seqlens;
    a.items = (int)items, a.rows = (int)rows, a.max_len = (int)max_len;
    a.k_heads = (int)k_heads, a.v_heads = (int)v_heads;
    a.scale = scale, a.eps = norm_eps;
    a.state_in = state_in, a.state_stride = state_stride, a.state_out = state_out;
    a.out = out, a.ldo = ldo;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = dtype == DB_DTYPE_F16 ? db::launch<__half>(a, workspace, s)
                                                : db::launch<__nv_bfloat16>(a, workspace, s);
    return db_cuda_status((int)e, "gated delta rule");
}

}  // extern "C"
