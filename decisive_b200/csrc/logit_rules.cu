// Rules on logits (db_logit_rules): penalties for repeated tokens, biases and a grammar mask, with
// the answer they lead to (best token, log-sum-exp).
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/decisive_b200.h"
#include "capi_internal.h"
#include "common.cuh"
#include "kernels.h"

namespace cg = cooperative_groups;

namespace db {
namespace {

constexpr int RULE_THREADS = 512, RULE_MAX_CTAS = 16, RULE_MAX_BIASES = 1024;
constexpr int RULE_MAX_SLICE = 49152;  // tokens of one CTA: their counters take 192 KB

struct RuleArgs {
    const void* logits;
    int64_t ld;
    int vocab, slice;
    const int32_t* history;
    int64_t ldh;
    const int32_t* history_lens;
    int history_cols;
    const float *repetition, *presence, *frequency;
    const int32_t* bias_ids;
    const float* bias_values;
    int biases;
    const uint32_t* mask;
    int64_t ldm;
    float* out;
    int64_t ldo;
    int32_t* best;
    float* lse;
};

// Running (largest value, its lowest index, sum of e^(value - largest)) of a set of tokens.
// A NaN makes the sum NaN and is never the largest value.
struct Stat {
    float top, sum;
    int at;
};
__device__ __forceinline__ Stat join(Stat a, Stat b) {
    Stat r;
    const bool b_wins = b.top > a.top || (b.top == a.top && b.at < a.at);
    r.top = b_wins ? b.top : a.top;
    r.at = b_wins ? b.at : a.at;
    // equal tops (both +inf among them) keep their sums as they are
    const float fa = a.top == r.top ? 1.f : exp2f((a.top - r.top) * 1.4426950408889634f);
    const float fb = b.top == r.top ? 1.f : exp2f((b.top - r.top) * 1.4426950408889634f);
    r.sum = a.sum * fa + b.sum * fb;
    return r;
}

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

// One row per cluster, a slice of the vocabulary per CTA; HBM bound: logits in, values out.  A
// token is looked up in detail only where a bit says that the history or a bias names it, so the
// stream itself costs a load, a mask test, an exponential and a store.  Counters live in shared
// memory and only those that the history names are ever touched (cleared, then counted): nothing of
// the vocabulary's size is initialised.  The CTAs' statistics meet in the first one's shared memory.
// VEC: logits per load (16 bytes), 1 where rows are not 16-byte aligned.
template <typename T, int VEC>
__global__ void __launch_bounds__(RULE_THREADS) logit_rules_kernel(RuleArgs a) {
    extern __shared__ __align__(16) uint32_t rule_smem[];
    __shared__ Stat warp_stat[RULE_THREADS / 32];
    __shared__ Stat cta_stat[RULE_MAX_CTAS];
    cg::cluster_group cluster = cg::this_cluster();
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, row = blockIdx.y;
    const int lo = blockIdx.x * a.slice, n = min(a.slice, a.vocab - lo);  // n may be <= 0 in the last CTAs
    const int words = a.slice / 32;
    uint32_t* seen = rule_smem;             // tokens of the slice that the history names
    uint32_t* biased = seen + words;        // ... that a bias names
    uint32_t* count = biased + words;       // [slice], valid where seen
    int32_t* ids = reinterpret_cast<int32_t*>(count + a.slice);
    float* values = reinterpret_cast<float*>(ids + a.biases);
    for (int i = tid; i < 2 * words; i += RULE_THREADS) seen[i] = 0;
    __syncthreads();
    const int32_t* history = a.history + (int64_t)row * a.ldh;
    const int length = a.history ? min(max(a.history_lens ? a.history_lens[row] : a.history_cols, 0), a.history_cols) : 0;
    for (int i = tid; i < length; i += RULE_THREADS) {
        const int c = (int)((unsigned)history[i] - (unsigned)lo);
        if ((unsigned)history[i] < (unsigned)a.vocab && (unsigned)c < (unsigned)a.slice) {
            count[c] = 0;
            atomicOr(&seen[c >> 5], 1u << (c & 31));
        }
    }
    for (int i = tid; i < a.biases; i += RULE_THREADS) {
        const int32_t id = a.bias_ids[(int64_t)row * a.biases + i];
        const int c = (unsigned)id < (unsigned)a.vocab ? id - lo : -1;
        ids[i] = c;
        values[i] = a.bias_values[(int64_t)row * a.biases + i];
        if ((unsigned)c < (unsigned)a.slice) atomicOr(&biased[c >> 5], 1u << (c & 31));
    }
    __syncthreads();
    for (int i = tid; i < length; i += RULE_THREADS) {
        const int c = (int)((unsigned)history[i] - (unsigned)lo);
        if ((unsigned)history[i] < (unsigned)a.vocab && (unsigned)c < (unsigned)a.slice) atomicAdd(&count[c], 1u);
    }
    __syncthreads();

    const float rho = a.repetition ? a.repetition[row] : 1.f;
    const float presence = a.presence ? a.presence[row] : 0.f, frequency = a.frequency ? a.frequency[row] : 0.f;
    const T* in = static_cast<const T*>(a.logits) + (int64_t)row * a.ld + lo;
    float* out = a.out + (int64_t)row * a.ldo + lo;
    const uint32_t* mask = a.mask ? a.mask + (int64_t)row * a.ldm + lo / 32 : nullptr;
    Stat mine = {-INFINITY, 0.f, 0x7fffffff};
    for (int c0 = tid * VEC; c0 < n; c0 += RULE_THREADS * VEC) {
        float x[VEC];
        if (VEC > 1 && c0 + VEC <= n) {
            const uint4 r = __ldcs(reinterpret_cast<const uint4*>(in + c0));
            const T* p = reinterpret_cast<const T*>(&r);
#pragma unroll
            for (int i = 0; i < VEC; ++i) x[i] = to_f32(p[i]);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) x[i] = c0 + i < n ? to_f32(in[c0 + i]) : -INFINITY;
        }
        const int shift = c0 & 31;
        const uint32_t bits = VEC == 32 ? 0xffffffffu : (1u << VEC) - 1;
        const uint32_t allowed = mask ? (mask[c0 >> 5] >> shift) & bits : bits;
        const uint32_t h = (seen[c0 >> 5] >> shift) & bits, w = (biased[c0 >> 5] >> shift) & bits;
        if (h | w) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                if (h >> i & 1) {
                    x[i] = x[i] > 0.f ? __fdiv_rn(x[i], rho) : __fmul_rn(x[i], rho);
                    x[i] = __fsub_rn(x[i], __fadd_rn(presence, __fmul_rn(frequency, (float)count[c0 + i])));
                }
                if (w >> i & 1)
                    for (int j = 0; j < a.biases; ++j)
                        if (ids[j] == c0 + i) x[i] = __fadd_rn(x[i], values[j]);
            }
        }
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            if (!(allowed >> i & 1)) x[i] = -INFINITY;
            top = fmaxf(top, x[i]);
        }
        if (VEC > 1 && c0 + VEC <= n) {
#pragma unroll
            for (int i = 0; i < VEC; i += 4)
                __stcs(reinterpret_cast<float4*>(out + c0 + i), make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]));
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (c0 + i < n) out[c0 + i] = x[i];
        }
        if (top > mine.top) {
            mine.sum = top == INFINITY ? mine.sum * 0.f : mine.sum * exp2f((mine.top - top) * 1.4426950408889634f);
            mine.top = top;
#pragma unroll
            for (int i = VEC - 1; i >= 0; --i)
                if (x[i] == top) mine.at = lo + c0 + i;
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            // the largest value counts 1 (+inf too), a token that is out 0, a NaN itself
            const float e = exp2f((x[i] - mine.top) * 1.4426950408889634f);
            mine.sum += x[i] == -INFINITY ? 0.f : x[i] == mine.top ? 1.f : e;
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        Stat other;
        other.top = __shfl_xor_sync(0xffffffffu, mine.top, o);
        other.sum = __shfl_xor_sync(0xffffffffu, mine.sum, o);
        other.at = __shfl_xor_sync(0xffffffffu, mine.at, o);
        // lower lane first on both sides, so the two halves of a pair agree to the bit
        mine = (tid & o) ? join(other, mine) : join(mine, other);
    }
    if ((tid & 31) == 0) warp_stat[tid >> 5] = mine;
    cluster.sync();  // also: the first CTA's shared memory is there to be written
    if (tid == 0) {
        Stat all = warp_stat[0];
        for (int i = 1; i < RULE_THREADS / 32; ++i) all = join(all, warp_stat[i]);
        *cluster.map_shared_rank(&cta_stat[cluster.block_rank()], 0) = all;
    }
    cluster.sync();
    if (cluster.block_rank() == 0 && tid == 0) {
        Stat all = cta_stat[0];
        for (int i = 1; i < (int)cluster.num_blocks(); ++i) all = join(all, cta_stat[i]);
        if (a.best) a.best[row] = all.top == -INFINITY ? -1 : all.at;
        // nothing allowed: log 0 = -inf (and NaN where a NaN was allowed)
        if (a.lse) a.lse[row] = all.top == -INFINITY ? (all.sum == 0.f ? -INFINITY : all.sum) : all.top + logf(all.sum);
    }
}

template <typename T>
cudaError_t launch(RuleArgs a, int rows, cudaStream_t stream) {
    constexpr int VEC = 16 / sizeof(T);
    const bool vec = !(((uintptr_t)a.logits | (uintptr_t)a.out) & 15) && !((a.ld * sizeof(T)) & 15) && !((a.ldo * 4) & 15);
    // CTAs per row: at least 2048 tokens each, all 16 for a vocabulary of 32 K tokens and more
    int ctas = 1;
    while (ctas < RULE_MAX_CTAS && (a.vocab + ctas - 1) / ctas > 2048) ctas *= 2;
    a.slice = ((a.vocab + ctas - 1) / ctas + 31) / 32 * 32;
    const size_t smem = (size_t)a.slice / 32 * 8 + (size_t)a.slice * 4 + (size_t)a.biases * 8;
    auto kernel = vec ? logit_rules_kernel<T, VEC> : logit_rules_kernel<T, 1>;
    static thread_local int ready_device[2] = {-1, -1};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (ready_device[vec] != dev) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
        ready_device[vec] = dev;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas, rows);
    cfg.blockDim = dim3(RULE_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {(unsigned)ctas, 1, 1};
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

}  // namespace
}  // namespace db

extern "C" int db_logit_rules(const void* logits, int dtype, int64_t ld, int64_t rows, int64_t vocab,
                              const int32_t* history, int64_t ldh, const int32_t* history_lens, int64_t history_cols,
                              const float* repetition, const float* presence, const float* frequency,
                              const int32_t* bias_ids, const float* bias_values, int64_t biases, const uint32_t* mask,
                              int64_t ldm, float* out, int64_t ldo, int32_t* best, float* lse, void* stream) {
    if (rows < 0 || rows > 65535 || vocab <= 0 || history_cols < 0 || history_cols >= ((int64_t)1 << 31) || biases < 0)
        return db_fail(DB_ERR_INVALID_ARGUMENT, "INVALID_ARGUMENT", "logit rules: bad shape");
    if (vocab > (int64_t)db::RULE_MAX_CTAS * db::RULE_MAX_SLICE)
        return db_fail(DB_ERR_UNSUPPORTED, "UNSUPPORTED", "logit rules: more than 786432 tokens");
    if (biases > db::RULE_MAX_BIASES)
        return db_fail(DB_ERR_UNSUPPORTED, "UNSUPPORTED", "logit rules: more than 1024 biases per row");
    if (dtype < DB_DTYPE_F32 || dtype > DB_DTYPE_BF16)
        return db_fail(DB_ERR_UNSUPPORTED, "UNSUPPORTED", "logit rules: logits are f32, f16 or bf16");
    if (rows == 0) return DB_OK;
    if (!logits || !out || ld < vocab || ldo < vocab || (mask && ldm < (vocab + 31) / 32) ||
        (history && ldh < history_cols) || (!history && history_lens) || (biases && (!bias_ids || !bias_values)))
        return db_fail(DB_ERR_INVALID_ARGUMENT, "INVALID_ARGUMENT", "logit rules: missing tensor or short row");
    if (static_cast<const void*>(out) == logits && (dtype != DB_DTYPE_F32 || ld != ldo))
        return db_fail(DB_ERR_INVALID_ARGUMENT, "INVALID_ARGUMENT", "logit rules: only f32 logits can be changed in place");
    db::RuleArgs a{};
    a.logits = logits, a.ld = ld, a.vocab = (int)vocab;
    a.history = history_cols ? history : nullptr, a.ldh = ldh, a.history_lens = history_lens,
    a.history_cols = (int)history_cols;
    a.repetition = repetition, a.presence = presence, a.frequency = frequency;
    a.bias_ids = bias_ids, a.bias_values = bias_values, a.biases = (int)biases;
    a.mask = mask, a.ldm = ldm;
    a.out = out, a.ldo = ldo, a.best = best, a.lse = lse;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = dtype == DB_DTYPE_F32   ? db::launch<float>(a, (int)rows, s)
                    : dtype == DB_DTYPE_F16 ? db::launch<__half>(a, (int)rows, s)
                                            : db::launch<__nv_bfloat16>(a, (int)rows, s);
    return db_cuda_status((int)e, "logit rules");
}
