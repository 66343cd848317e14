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
// T and P need no state: delta_prepare_kernel forms them for all chunks at once; delta_chunk_kernel then
// walks a sequence's chunks.
//
// Numerics.  The state has to keep f32's accuracy through f16 tensor products: k and q enter them exactly
// (bf16 rows as f16 after a power of two per row, which loses nothing within 2^-24 of the row's largest
// value; their lengths are applied afterwards as factors per token), and every f32 operand (S, R, U, T, P) as
// the sum of two f16 parts after a power of two per row: 22 bits.  lo x lo products are left out (2^-22).
// Decay sums are taken in f64: differences of f32 sums would lose what a slow decay has left.
constexpr int C = 64;                    // tokens per chunk
constexpr int BLOCKS = 10;               // 16 x 16 blocks of a lower triangle of 64
constexpr int TRI = BLOCKS * 256;        // halves of one triangle, in fragment order
constexpr int FACTORS = 5 * C + 4;       // floats per chunk and head: see Factor
// factors per token: R (times S k), O (times S q), U' (times U), rows of T, rows of P; then e^G_C
enum Factor { F_R = 0, F_O = C, F_U = 2 * C, F_T = 3 * C, F_P = 4 * C, F_END = 5 * C };

struct ChunkSpace {
    __half *k16, *q16;  // bf16 inputs: the rows as f16, [chunk ids][C][k_heads][D]; null for f16 inputs
    __half* tri;        // [chunk ids][v_heads][4][TRI]: T hi, T lo, P hi, P lo
    float* factor;      // [chunk ids][v_heads][FACTORS]
};

// Chunk ids: item b's chunks start at start_b / C + b, which leaves every item room for all of its chunks.
__host__ __device__ inline int64_t chunk_ids(int64_t rows, int64_t items) { return rows / C + items; }

size_t chunk_space(int64_t items, int64_t rows, int k_heads, int v_heads, bool copies, uint8_t* base, ChunkSpace* w) {
    const int64_t n = chunk_ids(rows, items);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        uint8_t* p = base ? base + at : nullptr;
        at += (bytes + 255) / 256 * 256;
        return p;
    };
    ChunkSpace s{};
    if (copies) {
        s.k16 = reinterpret_cast<__half*>(take((size_t)n * C * k_heads * D * 2));
        s.q16 = reinterpret_cast<__half*>(take((size_t)n * C * k_heads * D * 2));
    }
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
__device__ __forceinline__ void ldmatrix4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
// Byte offset of 16-byte piece c of row r in a tile of 256-byte rows (pieces permuted per row so that eight
// rows of one column of pieces lie on different banks).
__device__ __forceinline__ uint32_t tile_at(int r, int c) { return (uint32_t)(r * 256 + ((c ^ (r & 7)) << 4)); }

// 2^e that brings a largest magnitude m into [2^14, 2^15) (1 for 0, infinities and NaN), and 2^-e.
__device__ __forceinline__ float row_power(float m, float& back) {
    const int e = (int)((__float_as_uint(m) >> 23) & 0xff) - 127;
    const int k = m > 0.f && e < 128 ? min(max(14 - e, -126), 126) : 0;
    back = __uint_as_float((uint32_t)(127 - k) << 23);
    return __uint_as_float((uint32_t)(127 + k) << 23);
}
__device__ __forceinline__ float quad_max(float x) {
    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
    return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
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
    uint8_t k[C * 256], q[C * 256];  // f16 tiles
    float A[C * AP], T[C * AP], tmp[32 * 36];
    double G[C];
    float beta[C], rk[C], rq[C];
};

// T, P and the factors of one chunk, for one key head and the value heads that share it.
template <typename T>
__global__ void __launch_bounds__(PREP_THREADS) delta_prepare_kernel(DeltaArgs a, ChunkSpace w) {
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

    // rows into shared memory as f16, with their factors
    constexpr bool COPY = sizeof(T) == 2 && !std::is_same<T, __half>::value;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
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
                if (COPY) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            }
            float back = 1.f;
            uint4 y = raw[it];
            if (COPY) {
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
            if (c == 0) (which ? sh.rq : sh.rk)[r] = (a.eps >= 0.f ? rsqrtf(ss + a.eps) : 1.f) * (which ? a.scale : 1.f) * back;
        }
    }
    __syncthreads();

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

    const int group = a.v_heads / a.k_heads;
    for (int hv = hk * group; hv < (hk + 1) * group; ++hv) {
        __half* tri = w.tri + ((int64_t)id * a.v_heads + hv) * 4 * TRI;
        float* factor = w.factor + ((int64_t)id * a.v_heads + hv) * FACTORS;
        __syncthreads();  // the previous head's triangles have been read
        if (warp == 0) {
            double x[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int i = 2 * lane + j;
                const float gi = i < n ? a.g[(int64_t)(row0 + i) * a.ldg + hv] : 0.f;
                x[j] = gi < -1e4f ? -1e4 : (double)gi;  // e^-10000 = 0; -inf would make differences NaN
                sh.beta[i] = i < n ? a.beta[(int64_t)(row0 + i) * a.ldb + hv] : 0.f;
            }
            double sum = x[0] + x[1];
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const double y = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += y;
            }
            const double all = __shfl_sync(0xffffffffu, sum, 31);
            sh.G[2 * lane] = sum - x[1];
            sh.G[2 * lane + 1] = sum;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int i = 2 * lane + j;
                const double G = j ? sum : sum - x[1];
                const float e = expf((float)G);
                factor[F_R + i] = e * sh.rk[i];
                factor[F_O + i] = e * sh.rq[i];
                factor[F_U + i] = expf((float)(all - G)) * sh.rk[i];
            }
            if (lane == 0) factor[F_END] = expf((float)all);
        }
        __syncthreads();
        // A into shared memory, P to its place (the fragment of the block that a lane holds is what a lane of
        // the product P U takes)
        float p[8][4], ptop[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < 2 * warp + 2) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = warp * 16 + g + 8 * (i >> 1), c = 8 * j + 2 * t + (i & 1);
                    const float d = c <= r ? expf((float)(sh.G[r] - sh.G[c])) * sh.rk[c] : 0.f;
                    sh.A[r * AP + c] = c < r ? kk[j][i] * d * sh.rk[r] * sh.beta[r] : 0.f;
                    p[j][i] = c <= r ? qk[j][i] * d * sh.rq[r] : 0.f;
                    ptop[i >> 1] = fmaxf(ptop[i >> 1], fabsf(p[j][i]));
                }
            }
        auto store = [&](float (&x)[8][4], float top0, float top1, int which, int f) {
            float back[2];
            const float up[2] = {row_power(quad_max(top0), back[0]), row_power(quad_max(top1), back[1])};
            if (t == 0) {
                factor[f + warp * 16 + g] = back[0];
                factor[f + warp * 16 + 8 + g] = back[1];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j <= warp) {
                    uint4 h, l;
                    split2(x[2 * j][0] * up[0], x[2 * j][1] * up[0], h.x, l.x);
                    split2(x[2 * j + 1][0] * up[0], x[2 * j + 1][1] * up[0], h.y, l.y);
                    split2(x[2 * j][2] * up[1], x[2 * j][3] * up[1], h.z, l.z);
                    split2(x[2 * j + 1][2] * up[1], x[2 * j + 1][3] * up[1], h.w, l.w);
                    const int at = (warp * (warp + 1) / 2 + j) * 256 + lane * 8;
                    *reinterpret_cast<uint4*>(tri + which * TRI + at) = h;
                    *reinterpret_cast<uint4*>(tri + (which + 1) * TRI + at) = l;
                }
        };
        store(p, ptop[0], ptop[1], 2, F_P);
        __syncthreads();
        // (I + A)^-1, 16 x 16 blocks on the diagonal: lane c < 16 of warp b solves for column c of block b
        if (lane < 16) {
            const float* Ab = sh.A + (16 * warp) * AP + 16 * warp;
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = i == lane ? 1.f : 0.f;
#pragma unroll
            for (int i = 1; i < 16; ++i) {
                float s = 0.f;
#pragma unroll
                for (int j = 0; j < i; ++j) s = fmaf(Ab[i * AP + j], x[j], s);
                if (i != lane) x[i] = i > lane ? -s : 0.f;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) sh.T[(16 * warp + i) * AP + 16 * warp + lane] = x[i];
        }
        __syncthreads();
        // the block below two neighbours: -T11 A10 T00, first for 16 x 16 blocks, then for 32 x 32
        {
            const int pr = tid >> 6, c = tid & 15, r0 = ((tid >> 4) & 3) * 4, b0 = 32 * pr;
            float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                const float y = sh.T[(b0 + k) * AP + b0 + c];
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = fmaf(sh.A[(b0 + 16 + r0 + i) * AP + b0 + k], y, o[i]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) sh.tmp[(16 * pr + r0 + i) * 36 + c] = o[i];
            __syncthreads();
            float z[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                const float y = sh.tmp[(16 * pr + k) * 36 + c];
#pragma unroll
                for (int i = 0; i < 4; ++i) z[i] = fmaf(sh.T[(b0 + 16 + r0 + i) * AP + b0 + 16 + k], y, z[i]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) sh.T[(b0 + 16 + r0 + i) * AP + b0 + c] = -z[i];
            // the 16 x 16 blocks above the diagonal are zero
#pragma unroll
            for (int i = 0; i < 4; ++i) sh.T[(b0 + r0 + i) * AP + b0 + 16 + c] = 0.f;
        }
        __syncthreads();
        {
            const int c = lane, r0 = warp * 8;
            float o[8] = {};
#pragma unroll 4
            for (int k = 0; k < 32; k += 4) {
                float y[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] = sh.T[(k + j) * AP + c];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float4 x = *reinterpret_cast<const float4*>(&sh.A[(32 + r0 + i) * AP + k]);
                    o[i] = fmaf(x.w, y[3], fmaf(x.z, y[2], fmaf(x.y, y[1], fmaf(x.x, y[0], o[i]))));
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) sh.tmp[(r0 + i) * 36 + c] = o[i];
            __syncthreads();
            float z[8] = {};
#pragma unroll 4
            for (int k = 0; k < 32; k += 4) {
                float y[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] = sh.tmp[(k + j) * 36 + c];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float4 x = *reinterpret_cast<const float4*>(&sh.T[(32 + r0 + i) * AP + 32 + k]);
                    z[i] = fmaf(x.w, y[3], fmaf(x.z, y[2], fmaf(x.y, y[1], fmaf(x.x, y[0], z[i]))));
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) sh.T[(32 + r0 + i) * AP + c] = -z[i];
        }
        __syncthreads();
        float top[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < 2 * warp + 2) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = warp * 16 + g + 8 * (i >> 1), c = 8 * j + 2 * t + (i & 1);
                    p[j][i] = c <= r ? sh.T[r * AP + c] * sh.beta[c] : 0.f;
                    top[i >> 1] = fmaxf(top[i >> 1], fabsf(p[j][i]));
                }
            }
        store(p, top[0], top[1], 0, F_T);
    }
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// One buffered chunk of delta_chunk_kernel.
template <int WARPS>
struct Stage {
    uint8_t k[C * 256], q[C * 256];
    __half tri[4 * TRI];
    float factor[FACTORS];
    uint8_t v[C * WARPS * 32];  // this CTA's value features, 16 per warp
};

// Walks the chunks of one item and value head for 16 WARPS of the state's 128 value rows.  All products are
// formed transposed (rows = value features), so a warp keeps its 16 rows of the state in its accumulators,
// feeds them to the next product as they are, and never waits for another warp; what the rows share (k, q,
// T, P) is read from shared memory, the next chunk's while this one is worked on.
template <typename T, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, 1) delta_chunk_kernel(DeltaArgs a, ChunkSpace w) {
    extern __shared__ __align__(16) uint8_t chunk_smem[];
    Stage<WARPS>* stage = reinterpret_cast<Stage<WARPS>*>(chunk_smem);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int hv = blockIdx.y, b = blockIdx.z, hk = hv / (a.v_heads / a.k_heads);
    const int slice = blockIdx.x * 16 * WARPS, d0 = slice + 16 * warp;  // first value row of the CTA, the warp
    pdl_wait();
    pdl_trigger();
    int start, end;
    item_rows(a, b, start, end);
    const int chunks = (end - start + C - 1) / C;
    const int64_t id0 = start / C + b;

    float S[16][4];  // tile j: keys 8 j + 2 t, + 1 of value rows g (0, 1) and g + 8 (2, 3)
    const int64_t at = ((int64_t)hv * D + d0 + g) * D + 2 * t;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        float2 x = make_float2(0.f, 0.f), y = x;
        if (a.state_in) {
            const float* s = a.state_in + (int64_t)b * a.state_stride + at + 8 * j;
            x = *reinterpret_cast<const float2*>(s);
            y = *reinterpret_cast<const float2*>(s + 8 * D);
        }
        S[j][0] = x.x, S[j][1] = x.y, S[j][2] = y.x, S[j][3] = y.y;
    }

    constexpr int NT = 32 * WARPS;
    auto fetch = [&](int c) {
        Stage<WARPS>& st = stage[c & 1];
        const int row0 = start + c * C, n = min(C, end - row0);
        const int64_t id = id0 + c;
        const __half* k16 = w.k16 ? w.k16 + (id * C * a.k_heads + hk) * D
                                  : static_cast<const __half*>(a.k) + (int64_t)row0 * a.ldk + (int64_t)hk * D;
        const __half* q16 = w.q16 ? w.q16 + (id * C * a.k_heads + hk) * D
                                  : static_cast<const __half*>(a.q) + (int64_t)row0 * a.ldq + (int64_t)hk * D;
        const int64_t ldk = w.k16 ? (int64_t)a.k_heads * D : a.ldk, ldq = w.q16 ? (int64_t)a.k_heads * D : a.ldq;
        const uint32_t sk = smem_u32(st.k), sq = smem_u32(st.q), sv = smem_u32(st.v);
        for (int e = tid; e < C * 16; e += NT) {
            const int r = e >> 4, p = e & 15;
            const bool there = r < n;
            const int rr = there ? r : 0;
            cp_async16(sk + tile_at(r, p), k16 + rr * ldk + 8 * p, there);
            cp_async16(sq + tile_at(r, p), q16 + rr * ldq + 8 * p, there);
        }
        const T* v = static_cast<const T*>(a.v) + (int64_t)row0 * a.ldv + (int64_t)hv * D + slice;
        for (int e = tid; e < C * 2 * WARPS; e += NT) {
            const int r = e / (2 * WARPS), p = e % (2 * WARPS);
            const bool there = r < n;
            cp_async16(sv + r * WARPS * 32 + ((p ^ (r & (2 * WARPS - 1) & 7)) << 4), v + (there ? r : 0) * a.ldv + 8 * p, there);
        }
        const uint8_t* tri = reinterpret_cast<const uint8_t*>(w.tri + (id * a.v_heads + hv) * 4 * TRI);
        const uint32_t stri = smem_u32(st.tri);
        for (int e = tid; e < 4 * TRI * 2 / 16; e += NT) cp_async16(stri + 16 * e, tri + 16 * e, true);
        const uint8_t* f = reinterpret_cast<const uint8_t*>(w.factor + (id * a.v_heads + hv) * FACTORS);
        const uint32_t sf = smem_u32(st.factor);
        for (int e = tid; e < FACTORS / 4; e += NT) cp_async16(sf + 16 * e, f + 16 * e, true);
        cp_async_commit();
    };
    if (chunks > 0) fetch(0);
    for (int c = 0; c < chunks; ++c) {
        if (c + 1 < chunks) {
            fetch(c + 1);
            cp_async_wait<1>();
        } else {
            cp_async_wait<0>();
        }
        __syncthreads();
        const Stage<WARPS>& st = stage[c & 1];
        const uint32_t sk = smem_u32(st.k), sq = smem_u32(st.q), sv = smem_u32(st.v);
        const float* f = st.factor;

        // X = S [K; Q]^T: tiles 0-7 tokens of K, 8-15 of Q
        float X[16][4];
        float up[2], back[2];
        {
            float top[2] = {0.f, 0.f};
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                top[0] = fmaxf(top[0], fmaxf(fabsf(S[j][0]), fabsf(S[j][1])));
                top[1] = fmaxf(top[1], fmaxf(fabsf(S[j][2]), fabsf(S[j][3])));
#pragma unroll
                for (int i = 0; i < 4; ++i) X[j][i] = 0.f;
            }
            up[0] = row_power(quad_max(top[0]), back[0]);
            up[1] = row_power(quad_max(top[1]), back[1]);
        }
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            uint32_t h[4], l[4];
            split2(S[2 * s][0] * up[0], S[2 * s][1] * up[0], h[0], l[0]);
            split2(S[2 * s][2] * up[1], S[2 * s][3] * up[1], h[1], l[1]);
            split2(S[2 * s + 1][0] * up[0], S[2 * s + 1][1] * up[0], h[2], l[2]);
            split2(S[2 * s + 1][2] * up[1], S[2 * s + 1][3] * up[1], h[3], l[3]);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                uint32_t bb[4];
                ldmatrix4(bb, (j < 4 ? sk : sq) +
                                  tile_at(16 * (j & 3) + ((lane >> 4) << 3) + (lane & 7), 2 * s + ((lane >> 3) & 1)));
                mma16816(X[2 * j], l, bb[0], bb[1]);
                mma16816(X[2 * j + 1], l, bb[2], bb[3]);
                mma16816(X[2 * j], h, bb[0], bb[1]);
                mma16816(X[2 * j + 1], h, bb[2], bb[3]);
            }
        }
        // R = V - e^G S k, in place of the K half
        float top[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            // V^T fragments of tokens 16 j .. + 15: value rows 0-7, 8-15 of tokens 0-7, then of 8-15
            uint32_t vv[4];
            const int r = 16 * j + ((lane >> 4) << 3) + (lane & 7), p = 2 * warp + ((lane >> 3) & 1);
            ldmatrix4t(vv, sv + r * WARPS * 32 + ((p ^ (r & (2 * WARPS - 1) & 7)) << 4));
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                const float2 ff = *reinterpret_cast<const float2*>(&f[F_R + 16 * j + 8 * hh + 2 * t]);
                float (&x)[4] = X[2 * j + hh];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t word = vv[2 * hh + (i >> 1)];
                    const unsigned short u = (unsigned short)(i & 1 ? word >> 16 : word & 0xffffu);
                    x[i] = fmaf(-((i & 1) ? ff.y : ff.x), x[i] * back[i >> 1], to_f32(*reinterpret_cast<const T*>(&u)));
                    top[i >> 1] = fmaxf(top[i >> 1], fabsf(x[i]));
                }
            }
        }
        float ru[2], rb[2];
        ru[0] = row_power(quad_max(top[0]), rb[0]);
        ru[1] = row_power(quad_max(top[1]), rb[1]);
        uint32_t ah[4][4], al[4][4];
        auto split_rows = [&](const float (&x0)[4], const float (&x1)[4], float u0, float u1, uint32_t (&h)[4], uint32_t (&l)[4]) {
            split2(x0[0] * u0, x0[1] * u0, h[0], l[0]);
            split2(x0[2] * u1, x0[3] * u1, h[1], l[1]);
            split2(x1[0] * u0, x1[1] * u0, h[2], l[2]);
            split2(x1[2] * u1, x1[3] * u1, h[3], l[3]);
        };
#pragma unroll
        for (int s = 0; s < 4; ++s) split_rows(X[2 * s], X[2 * s + 1], ru[0], ru[1], ah[s], al[s]);
        // Y += (a triangle of T or P) applied to the rows in ah, al
        auto triangle = [&](float (&Y)[8][4], int which) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) Y[j][i] = 0.f;
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int j = s; j < 4; ++j) {
                    const int blk = (j * (j + 1) / 2 + s) * 256 + lane * 8;
                    const uint4 bh = *reinterpret_cast<const uint4*>(st.tri + which * TRI + blk);
                    const uint4 bl = *reinterpret_cast<const uint4*>(st.tri + (which + 1) * TRI + blk);
                    mma16816(Y[2 * j], al[s], bh.x, bh.y);
                    mma16816(Y[2 * j + 1], al[s], bh.z, bh.w);
                    mma16816(Y[2 * j], ah[s], bl.x, bl.y);
                    mma16816(Y[2 * j + 1], ah[s], bl.z, bl.w);
                    mma16816(Y[2 * j], ah[s], bh.x, bh.y);
                    mma16816(Y[2 * j + 1], ah[s], bh.z, bh.w);
                }
        };
        float U[8][4];
        triangle(U, 0);
        float utop[2] = {0.f, 0.f}, wtop[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float2 ft = *reinterpret_cast<const float2*>(&f[F_T + 8 * j + 2 * t]);
            const float2 fu = *reinterpret_cast<const float2*>(&f[F_U + 8 * j + 2 * t]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                U[j][i] *= rb[i >> 1] * ((i & 1) ? ft.y : ft.x);
                X[j][i] = U[j][i] * ((i & 1) ? fu.y : fu.x);  // what the state takes, over k
                utop[i >> 1] = fmaxf(utop[i >> 1], fabsf(U[j][i]));
                wtop[i >> 1] = fmaxf(wtop[i >> 1], fabsf(X[j][i]));
            }
        }
        // the state: S <- e^G_C S + U'^T K, eight tiles of keys at a time
        float wu[2], wb[2];
        wu[0] = row_power(quad_max(wtop[0]), wb[0]);
        wu[1] = row_power(quad_max(wtop[1]), wb[1]);
#pragma unroll
        for (int s = 0; s < 4; ++s) split_rows(X[2 * s], X[2 * s + 1], wu[0], wu[1], ah[s], al[s]);
        const float decay = f[F_END];
#pragma unroll
        for (int part = 0; part < 4; ++part) {
            float Y[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) Y[j][i] = 0.f;
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    // K^T: keys 32 part + 16 j .. + 15 of tokens 16 s .. + 15
                    uint32_t bb[4];
                    ldmatrix4t(bb, sk + tile_at(16 * s + ((lane >> 3) & 1) * 8 + (lane & 7), 4 * part + 2 * j + (lane >> 4)));
                    mma16816(Y[2 * j], al[s], bb[0], bb[1]);
                    mma16816(Y[2 * j + 1], al[s], bb[2], bb[3]);
                    mma16816(Y[2 * j], ah[s], bb[0], bb[1]);
                    mma16816(Y[2 * j + 1], ah[s], bb[2], bb[3]);
                }
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) S[4 * part + j][i] = fmaf(S[4 * part + j][i], decay, Y[j][i] * wb[i >> 1]);
        }
        // O = e^G S0 q + P U
        float uu[2], ub[2];
        uu[0] = row_power(quad_max(utop[0]), ub[0]);
        uu[1] = row_power(quad_max(utop[1]), ub[1]);
#pragma unroll
        for (int s = 0; s < 4; ++s) split_rows(U[2 * s], U[2 * s + 1], uu[0], uu[1], ah[s], al[s]);
        float O[8][4];
        triangle(O, 2);
        const int row0 = start + c * C, n = end - row0;
        T* out = static_cast<T*>(a.out) + (int64_t)row0 * a.ldo + (int64_t)hv * D + d0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float2 fo = *reinterpret_cast<const float2*>(&f[F_O + 8 * j + 2 * t]);
            const float2 fp = *reinterpret_cast<const float2*>(&f[F_P + 8 * j + 2 * t]);
            uint32_t word[2];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = fmaf((i & 1) ? fo.y : fo.x, X[8 + j][i] * back[i >> 1],
                                     O[j][i] * (ub[i >> 1] * ((i & 1) ? fp.y : fp.x)));
                T y;
                from_f32(x, y);
                const uint32_t u = *reinterpret_cast<const unsigned short*>(&y);
                if (i & 1) word[i >> 1] |= u << 16; else word[i >> 1] = u;
            }
            // transposed: token g, value rows 2 t, 2 t + 1 of either half
            uint32_t lo8, hi8;
            asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(lo8) : "r"(word[0]));
            asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(hi8) : "r"(word[1]));
            if (8 * j + g < n) {
                T* dst = out + (int64_t)(8 * j + g) * a.ldo + 2 * t;
                *reinterpret_cast<uint32_t*>(dst) = lo8;
                *reinterpret_cast<uint32_t*>(dst + 8) = hi8;
            }
        }
        __syncthreads();  // the stage may be filled again
    }
    if (a.state_out) {
        float* s = a.state_out + (int64_t)b * a.v_heads * D * D + at;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            *reinterpret_cast<float2*>(s + 8 * j) = make_float2(S[j][0], S[j][1]);
            *reinterpret_cast<float2*>(s + 8 * j + 8 * D) = make_float2(S[j][2], S[j][3]);
        }
    }
}

// Up to this many tokens per item the recurrence is faster than a chunk.
constexpr int STEP_TOKENS = DB_DELTA_STEP_TOKENS;

template <typename T, int WARPS>
cudaError_t launch_chunks(const DeltaArgs& a, const ChunkSpace& w, cudaStream_t stream) {
    auto kernel = delta_chunk_kernel<T, WARPS>;
    const int smem = 2 * sizeof(Stage<WARPS>);
    cudaError_t e = db_set_max_smem(reinterpret_cast<const void*>(kernel), smem);
    if (e != cudaSuccess) return e;
    return db_launch_pdl(kernel, dim3(D / (16 * WARPS), a.v_heads, a.items), dim3(32 * WARPS), smem, stream, a, w);
}

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
    e = db_launch_pdl(delta_prepare_kernel<T>, dim3((unsigned)chunk_ids(a.rows, a.items), a.k_heads), dim3(PREP_THREADS),
                      sizeof(PrepShared), stream, a, w);
    if (e != cudaSuccess) return e;
    // a head per CTA where heads fill the SMs, else half a head
    return a.v_heads * a.items >= db_num_sms() ? launch_chunks<T, 8>(a, w, stream) : launch_chunks<T, 4>(a, w, stream);
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
        v_heads > 65535 || v_heads % k_heads || (!cu_seqlens && rows != items * max_len) || max_len > rows)
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
    if (state_in && state_in == state_out && items > 1 && state_stride != v_heads * 128 * 128)
        return db_fail(DB_ERR_INVALID_ARGUMENT, "INVALID_ARGUMENT",
                       "gated delta rule: a state shared by several items cannot be updated in place");
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
