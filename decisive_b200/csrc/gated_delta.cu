// The gated delta rule (db_gated_delta): per sequence and value head a state S [128 value, 128 key]
// in f32 and, token by token,
//   S <- e^g S;  u = beta (v - S k);  S <- S + u k^T;  o = S q
// with k and q divided by their lengths (norm_eps >= 0) and q times `scale`.
#include <cuda_bf16.h>

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

template <typename T>
cudaError_t launch(const DeltaArgs& a, void* workspace, cudaStream_t stream) {
    (void)workspace;
    const dim3 grid(D / (STEP_ROWS * STEP_WARPS), a.v_heads, a.items);
    return db_launch_pdl(delta_step_kernel<T>, grid, dim3(32 * STEP_WARPS), 0, stream, a);
}

}  // namespace
}  // namespace db

extern "C" {

size_t db_gated_delta_workspace_bytes(int64_t items, int64_t rows, int64_t max_len, int64_t k_heads, int64_t v_heads) {
    (void)items, (void)rows, (void)max_len, (void)k_heads, (void)v_heads;
    return 0;
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
