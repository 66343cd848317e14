// Rules on logits (db_logit_rules): penalties for repeated tokens, biases and a grammar mask, with
// the answer they lead to (best token, log-sum-exp).
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <utility>

#include "../../include/decisive_b200.h"
#include "capi_internal.h"
#include "common.cuh"
#include "kernels.h"

namespace cg = cooperative_groups;

namespace db {
namespace {

constexpr int RULE_THREADS = 512, RULE_MAX_CTAS = 16, RULE_MAX_BIASES = 1024;
constexpr float LOG2E = 1.4426950408889634f;
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
    int narrow;  // 16-bit counters
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

// 2^x on the special-function unit
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The statistics of a warp's lanes, in every lane.
__device__ __forceinline__ Stat join_lanes(Stat mine) {
    Stat r;
    r.top = mine.top;
#pragma unroll
    for (int o = 16; o; o >>= 1) r.top = fmaxf(r.top, __shfl_xor_sync(0xffffffffu, r.top, o));
    // equal tops (both infinities among them) keep their sums as they are
    r.sum = mine.sum * (mine.top == r.top ? 1.f : ex2((mine.top - r.top) * LOG2E));
#pragma unroll
    for (int o = 16; o; o >>= 1) r.sum += __shfl_xor_sync(0xffffffffu, r.sum, o);
    r.at = (int)__reduce_min_sync(0xffffffffu, (unsigned)(mine.top == r.top ? mine.at : 0x7fffffff));
    return r;
}

// One row per cluster, every n-th stripe of 4096 tokens per CTA (common tokens have low ids: whole slices would
// leave the first CTA most of the history); HBM bound: logits in, values out.  The stream itself
// costs a load, a mask test, an exponential and a store, for 8 tokens of a lane at a time; the tokens that the
// history or a bias names are left out of it and taken afterwards from a list in the order of their ids, one
// to a lane (handled inside the stream, a few lanes of nearly every warp would hold up the others).
// Counters live in shared memory, 16 bits each while the history has fewer tokens than that.  The CTAs'
// statistics meet in the first one's shared memory.
// VEC: rows start on 16-byte boundaries.
constexpr int RULE_STEP = 8;                         // tokens of a lane at a time
constexpr int STRIPE = RULE_THREADS * RULE_STEP;     // tokens of a CTA at a time

// x added to a running statistic; -inf adds nothing
__device__ __forceinline__ void add_one(Stat& s, float x, int id) {
    Stat one;
    one.top = x == x ? x : -INFINITY;
    one.sum = x != x ? x : x == -INFINITY ? 0.f : 1.f;
    one.at = one.top == -INFINITY ? 0x7fffffff : id;
    s = join(s, one);
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(RULE_THREADS, 3) logit_rules_kernel(RuleArgs a) {
    extern __shared__ __align__(16) uint32_t rule_smem[];
    __shared__ Stat warp_stat[RULE_THREADS / 32];
    __shared__ Stat cta_stat[RULE_MAX_CTAS];
    __shared__ int warp_count[RULE_THREADS / 32];
    constexpr int WARPS = RULE_THREADS / 32;
    cg::cluster_group cluster = cg::this_cluster();
    auto started = cluster.barrier_arrive();  // waited for before another CTA's shared memory is written
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31, row = blockIdx.y;
    const int rank = blockIdx.x, ctas = gridDim.x;
    // local token c is token id_of(c); stripes past the vocabulary are empty
    auto id_of = [&](int c) { return ((c / STRIPE) * ctas + rank) * STRIPE + c % STRIPE; };
    const int words = a.slice / 32;
    uint32_t* seen = rule_smem;             // the CTA's tokens that the history names
    uint32_t* biased = seen + words;        // ... that a bias names
    uint32_t* count = biased + words;       // counters, two to a word where they have 16 bits
    const int two = a.narrow, counters = a.slice >> two;
    int32_t* ids = reinterpret_cast<int32_t*>(count + counters);
    float* values = reinterpret_cast<float*>(ids + a.biases);
    // a step's logits are on their way while the one before is worked on, the first while the history is counted
    constexpr int LOADS = RULE_STEP * sizeof(T) / 16, EACH = 16 / sizeof(T);
    const T* in = static_cast<const T*>(a.logits) + (int64_t)row * a.ld;
    uint4 ahead[LOADS];
    auto load = [&](int c) {
        if (VEC && c + RULE_STEP <= a.vocab)
#pragma unroll
            for (int k = 0; k < LOADS; ++k) ahead[k] = __ldcs(reinterpret_cast<const uint4*>(in + c) + k);
    };
    load(rank * STRIPE + tid * RULE_STEP);
    for (int i = tid; i < (2 * words + counters) / 4; i += RULE_THREADS) reinterpret_cast<uint4*>(seen)[i] = make_uint4(0, 0, 0, 0);
    const int32_t* history = a.history + (int64_t)row * a.ldh;
    const int length = a.history ? min(max(a.history_lens ? a.history_lens[row] : a.history_cols, 0), a.history_cols) : 0;
    __syncthreads();
    for (int i = tid; i < length; i += RULE_THREADS) {
        const int32_t id = history[i];
        const unsigned stripe = (unsigned)id / STRIPE, c = stripe / ctas * STRIPE + (unsigned)id % STRIPE;
        if ((unsigned)id < (unsigned)a.vocab && stripe % ctas == rank) {
            atomicAdd(&count[c >> two], two && (c & 1) ? 65536u : 1u);
            atomicOr(&seen[c >> 5], 1u << (c & 31));
        }
    }
    for (int i = tid; i < a.biases; i += RULE_THREADS) {
        const int32_t id = a.bias_ids[(int64_t)row * a.biases + i];
        const unsigned stripe = (unsigned)id / STRIPE;
        const int c = (unsigned)id < (unsigned)a.vocab && stripe % ctas == rank ? (int)(stripe / ctas * STRIPE + (unsigned)id % STRIPE) : -1;
        ids[i] = c;
        values[i] = a.bias_values[(int64_t)row * a.biases + i];
        if (c >= 0) atomicOr(&biased[c >> 5], 1u << (c & 31));
    }
    __syncthreads();

    float* out = a.out + (int64_t)row * a.ldo;
    const uint32_t* mask = a.mask ? a.mask + (int64_t)row * a.ldm : nullptr;
    Stat mine = {-INFINITY, 0.f, 0x7fffffff};
    for (int c0 = tid * RULE_STEP, v0 = rank * STRIPE + c0; v0 < a.vocab; c0 += STRIPE, v0 += ctas * STRIPE) {
        const bool whole = VEC && v0 + RULE_STEP <= a.vocab;
        float x[RULE_STEP];
        if (whole) {
#pragma unroll
            for (int k = 0; k < LOADS; ++k) {
                const T* p = reinterpret_cast<const T*>(&ahead[k]);
#pragma unroll
                for (int i = 0; i < EACH; ++i) x[k * EACH + i] = to_f32(p[i]);
            }
            load(v0 + ctas * STRIPE);
        } else {
#pragma unroll
            for (int i = 0; i < RULE_STEP; ++i) x[i] = v0 + i < a.vocab ? to_f32(in[v0 + i]) : -INFINITY;
        }
        const int word = c0 >> 5, shift = c0 & 31;
        const uint32_t named = seen[word] | biased[word];
        const uint32_t allowed = (mask ? mask[v0 >> 5] & ~named : ~named) >> shift;
        const uint32_t left = (named >> shift) & 0xffu;
        float top = -INFINITY;
        // a named token's logit is written as it came (the logits may be changed in place) and again when its rules have run:
        // lanes that hold one then store like the others (93 -> 89 us for 256 rows with 1000 tokens of history)
        const uint32_t shown = allowed | left;
#pragma unroll
        for (int i = 0; i < RULE_STEP; ++i) x[i] = (shown >> i & 1) ? x[i] : -INFINITY;
        if (whole) {
#pragma unroll
            for (int i = 0; i < RULE_STEP; i += 4)
                __stcs(reinterpret_cast<float4*>(out + v0 + i), make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]));
        } else {
#pragma unroll
            for (int i = 0; i < RULE_STEP; ++i)
                if (v0 + i < a.vocab) out[v0 + i] = x[i];
        }
        if (left) {
#pragma unroll
            for (int i = 0; i < RULE_STEP; ++i) x[i] = (left >> i & 1) ? -INFINITY : x[i];
        }
#pragma unroll
        for (int i = 0; i < RULE_STEP; ++i) top = fmaxf(top, x[i]);
        if (top > mine.top) {
            mine.sum = top == INFINITY ? mine.sum * 0.f : mine.sum * ex2((mine.top - top) * LOG2E);
            mine.top = top;
            int at = 0;
#pragma unroll
            for (int i = RULE_STEP - 1; i >= 0; --i) at = x[i] == top ? i : at;
            mine.at = v0 + at;
        }
        if (fabsf(mine.top) < 1e4f) {
            const float base = mine.top * LOG2E;  // its rounding is a common factor: 1e4 x 2^-24 at most
#pragma unroll
            for (int i = 0; i < RULE_STEP; ++i) mine.sum += ex2(fmaf(x[i], LOG2E, -base));
        } else {
#pragma unroll
            for (int i = 0; i < RULE_STEP; ++i)
                mine.sum += x[i] != x[i] ? x[i] : x[i] == mine.top ? (mine.top == -INFINITY ? 0.f : 1.f) : ex2((x[i] - mine.top) * LOG2E);
        }
    }

    // the named tokens: their places in the order of ids by a scan over the words' bit counts, then one to a lane
    int bits = 0;
    const int each = (words + RULE_THREADS - 1) / RULE_THREADS, w0 = tid * each, w1 = min(w0 + each, words);
    for (int i = w0; i < w1; ++i) bits += __popc(seen[i] | biased[i]);
    int place = bits;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const int y = __shfl_up_sync(0xffffffffu, place, o);
        if (lane >= o) place += y;
    }
    if (lane == 31) warp_count[tid >> 5] = place;
    __syncthreads();
    int total = 0;
    for (int i = 0; i < WARPS; ++i) {
        if (i == (tid >> 5)) place += total;
        total += warp_count[i];
    }
    place -= bits;
    int32_t* list = reinterpret_cast<int32_t*>(values + a.biases);  // RULE_THREADS entries at a time
    const float rho = a.repetition ? a.repetition[row] : 1.f;
    const float presence = a.presence ? a.presence[row] : 0.f, frequency = a.frequency ? a.frequency[row] : 0.f;
    for (int from = 0; from < total; from += RULE_THREADS) {
        if (from) __syncthreads();  // the list has been read
        int at = place;
        if (place < from + RULE_THREADS && place + bits > from)
            for (int i = w0; i < w1; ++i)
                for (uint32_t rest = seen[i] | biased[i]; rest; rest &= rest - 1, ++at)
                    if (at >= from && at < from + RULE_THREADS) list[at - from] = 32 * i + __ffs(rest) - 1;
        __syncthreads();
        if (from + tid >= total) continue;
        const int c = list[tid], id = id_of(c);
        float y = to_f32(in[id]);
        if (seen[c >> 5] >> (c & 31) & 1) {
            const uint32_t pair = count[c >> two], times = two ? (c & 1 ? pair >> 16 : pair & 0xffffu) : pair;
            y = y > 0.f ? __fdiv_rn(y, rho) : __fmul_rn(y, rho);
            y = __fsub_rn(y, __fadd_rn(presence, __fmul_rn(frequency, (float)times)));
        }
        if (biased[c >> 5] >> (c & 31) & 1)
            for (int j = 0; j < a.biases; ++j)
                if (ids[j] == c) y = __fadd_rn(y, values[j]);
        if (mask && !(mask[id >> 5] >> (id & 31) & 1)) y = -INFINITY;
        out[id] = y;
        add_one(mine, y, id);
    }
    mine = join_lanes(mine);
    if (lane == 0) warp_stat[tid >> 5] = mine;
    __syncthreads();
    cluster.barrier_wait(std::move(started));
    const Stat none = {-INFINITY, 0.f, 0x7fffffff};
    if (tid < 32) {
        const Stat all = join_lanes(lane < WARPS ? warp_stat[lane] : none);
        if (lane == 0) *cluster.map_shared_rank(&cta_stat[cluster.block_rank()], 0) = all;
    }
    // the others are done once theirs is on its way; the first one waits for all
    auto written = cluster.barrier_arrive();
    if (cluster.block_rank() != 0) return;
    cluster.barrier_wait(std::move(written));
    if (tid < 32) {
        const Stat all = join_lanes(lane < (int)cluster.num_blocks() ? cta_stat[lane] : none);
        if (lane == 0) {
            if (a.best) a.best[row] = all.top == -INFINITY ? -1 : all.at;
            // nothing allowed: log 0 = -inf (and NaN where a NaN was allowed)
            if (a.lse) a.lse[row] = all.top == -INFINITY ? (all.sum == 0.f ? -INFINITY : all.sum) : all.top + logf(all.sum);
        }
    }
}

template <typename T>
cudaError_t launch(RuleArgs a, int rows, cudaStream_t stream) {
    const bool vec = !(((uintptr_t)a.logits | (uintptr_t)a.out) & 15) && !((a.ld * sizeof(T)) & 15) && !((a.ldo * 4) & 15);
    // CTAs per row: for few rows one per stripe, up to 16; for many only as many as fill the SMs with three
    // each, so that a CTA's fixed work is spread over more tokens (64 rows of 151936 tokens, 8 CTAs each: 31 us; with six
    // to an SM, 16 CTAs each: 37 us)
    const int stripes = (a.vocab + STRIPE - 1) / STRIPE, fill = 3 * db_num_sms();
    int ctas = 1;
    while (ctas < RULE_MAX_CTAS && ctas < stripes && (stripes > ctas * (RULE_MAX_SLICE / 2 / STRIPE) || rows * ctas < fill)) ctas *= 2;
    a.slice = (stripes + ctas - 1) / ctas * STRIPE;
    a.narrow = a.history_cols < 65536;
    const size_t smem = (size_t)a.slice / 32 * 8 + (size_t)(a.slice >> a.narrow) * 4 + (size_t)a.biases * 8 + RULE_THREADS * 4;
    auto kernel = vec ? logit_rules_kernel<T, true> : logit_rules_kernel<T, false>;
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
