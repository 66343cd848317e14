// Attention over the 8-bit cache for many query rows (a chunk of a prompt), on the tcgen05 tensor cores.
//
// One CTA = 128 query rows of one kv head (token n / group, head n % group: neighbouring tokens share every key
// tile), one row per lane of tensor memory; keys in tiles of one block (64), one pass.  Even and odd tiles go to two
// softmax warpgroups, each with its own running maximum, sum and accumulator, joined at the end, so the tensor
// pipe always holds two independent chains.  Per tile
//   S = Q K^T (codes as exact f16),  P = 2^(S c - m),  O += P V (codes as exact f16)
// Six warps turn codes into f16 tiles in shared memory, in the order in which the MMAs take them; a value page is
// stored [128][64 tokens], which is already the K-major operand.  P stays in tensor memory: it overwrites S
// and is the A operand of the second product, as two f16 parts, 22 bits (one f16 would change one bf16 output in 15).
// Where scales go: a key block's into the exponent's factor, a value block's into P, relative to the accumulator's unit, a
// power of two of its warpgroup's; the row sum is taken back by the inverse.  The unit starts at 2 to 4 times the first
// block's value scale and moves, with the accumulator, to a block whose scale is above it or below 2^-6 of it, so the
// largest P lie far inside f16's normal range; a row depends only on what it sees, because the accumulator's factors are
// powers of two.  The unit stays above 2^-80 of the largest so far (the accumulator must not overflow): under a block 2^80 times as large,
// values end at 2^-100 of that block's.  The maximum moves only when a tile raises it by more than 4 (log2), so accumulators
// are rarely rescaled, and f16's subnormals begin 2^-23 below the maximum as a rule, 2^-19 at the least: weak keys add up.
//
// Warps: 0-3, 14 and 15 conversion, 4-7 softmax of even tiles, 8-11 of odd tiles, 12 and 13 MMA issue for even and odd
// tiles (one issuer for both was the kernel's bound: 3600 of 6600 cycles per pair of tiles), 12 tensor memory.
// Latency bound: each chain hands S, P and O from role to role, and two chains fill the gaps only in part; a CTA takes an
// SM whole (shared memory, tensor memory), so 2000 rows of 8 kv heads are one round of 128 CTAs.  B200, 1000 rows after 7000
// keys, 16 / 8 heads: 149 us, f16 and bf16 (412 TFLOP/s, 25% of the dense f16 rate; P's second part is a third of the
// products and not counted).
// Tensor memory (512 columns): S / P of (parity, slot) at 128 parity + 64 slot, O even 256-383, O odd 384-511.
#include <float.h>

#include "kv8.cuh"
#include "capi_internal.h"
#include "kernels.h"
#include "tc_chain.cuh"

namespace db {
namespace {

using chain::tie32;
using chain::warp_wait;

constexpr int D = KV8_D, BLK = KV8_BLK;
constexpr int ROWS = 128, THREADS = 512, CONVERTERS = 6;
constexpr int STAGES = 10, STAGE = BLK * D * 2;  // f16 tiles of one block's keys or values
constexpr int Q_BYTES = ROWS * D * 2, Q_HALF = Q_BYTES / 2, K_HALF = STAGE / 2;
constexpr int INFO = 16;                         // tiles whose scales are kept at a time
constexpr uint32_t TM_O = 256;
constexpr uint64_t DRAIN_NS = 100000000ull;

enum Bar { FULL = 0, EMPTY = FULL + STAGES, S_FULL = EMPTY + STAGES, P_FULL = S_FULL + 4, PV_DONE = P_FULL + 4,
           JOIN = PV_DONE + 4, MMA_DONE, END = MMA_DONE + 2, BARS };

constexpr float SLACK = 4.f;     // how far (log2) a tile may lie above the running maximum
constexpr int SHIFT = 11;        // P of the maximum is 2^SHIFT (value scale / unit), so of a key below 2^15
constexpr int NO_SCALE = -1000;  // a value scale that moves no unit
constexpr int LEAST = -40;       // P this far down is 0 in both parts
struct Info {
    float ks;      // key scale
    int e;         // the value scale is 2^e f, 1 <= f < 2; NO_SCALE: 0 (its block adds nothing) or not finite
    float lf, inv; // log2 f and 1 / f (NaN where the scale is not finite)
    int there;
};
struct Shared {
    uint64_t bars[BARS];
    Info info[INFO];
    float row_factor[ROWS];
    float join_m[2][ROWS], join_l[2][ROWS];
    int join_unit[2][ROWS];
    uint32_t tmem;
    int abort;
    uint32_t tail_v;                // bf16: the open block's largest value (its bits)
    alignas(16) float key_up[BLK], key_back[BLK];  // bf16: the open block's keys' powers of two
    int odd;                        // the open block has values that are not finite
};
constexpr int SMEM = 1024 + Q_BYTES + STAGES * STAGE + sizeof(Shared);
static_assert(SMEM <= 232448, "shared memory");

// 2^e that brings a largest magnitude m to [2^7, 2^8), the codes' own size (1 for 0); back = 2^-e.
__device__ __forceinline__ float code_power(float m, float& back) {
    const int e = (int)((__float_as_uint(m) >> 23) & 0xff) - 127;
    const int k = m > 0.f ? min(max(7 - e, -126), 126) : 0;
    back = __uint_as_float((uint32_t)(127 - k) << 23);
    return __uint_as_float((uint32_t)(127 + k) << 23);
}
// 2^n, 0 below f32's normal range (n <= 127)
__device__ __forceinline__ float power2(int n) { return n < -126 ? 0.f : __uint_as_float((uint32_t)(127 + n) << 23); }
__device__ __forceinline__ void sts128u(uint8_t* base, uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    *reinterpret_cast<uint4*>(base + at) = make_uint4(a, b, c, d);
}

// One row's softmax step on a tile's 64 scores: moves the maximum m (and l) if the tile raises it by more than SLACK, writes
// P = 2^(S scale + shift - m) over S as the operand (32 keys to 32 columns: 16 of first parts, 16 of second), returns
// its sum.  MASKED: only keys 0 .. seen count; a scale of 0 or NaN must not reach the others.
// PT: the type of P's parts.
template <bool MASKED, typename PT = __half>
__device__ __forceinline__ float soften(uint32_t (&r)[2][32], int seen, float scale, float shift, float& m, float& l, float& move,
                                        uint32_t s_tm) {
    if (MASKED) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (32 * c + i > seen) r[c][i] = __float_as_uint(-INFINITY);
    }
    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < 32; ++i) mx[i & 3] = fmaxf(mx[i & 3], __uint_as_float(r[c][i]));
    const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
    const float mt = top == -INFINITY ? top : top * scale;
    if (mt > m + SLACK) {  // (the first keys: from -inf)
        move = ex2(m - mt);
        m = mt;
        l *= move;
    }
    const float add = shift - (m == -INFINITY ? 0.f : m);
    const uint64_t scale2 = f2_pack(__float_as_uint(scale), __float_as_uint(scale)), add2 = f2_pack(__float_as_uint(add), __float_as_uint(add));
    const uint64_t minus = f2_pack(0xbf800000u, 0xbf800000u);
    uint64_t sum[2] = {0, 0};
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        uint32_t pk[32];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint64_t e = f2_fma(f2_pack(r[c][2 * i], r[c][2 * i + 1]), scale2, add2);
            float x = ex2(f2_lo(e)), y = ex2(f2_hi(e));
            if (MASKED) {
                if (32 * c + 2 * i > seen) x = 0.f;
                if (32 * c + 2 * i + 1 > seen) y = 0.f;
            }
            const uint64_t xy = f2_pack(__float_as_uint(x), __float_as_uint(y));
            sum[i & 1] = f2_add(sum[i & 1], xy);
            pk[i] = pack2<PT>(x, y);
            const uint64_t h = f2_pack(__float_as_uint(from_bits<PT>(pk[i] & 0xffffu)), __float_as_uint(from_bits<PT>(pk[i] >> 16)));
            const uint64_t left = f2_fma(h, minus, xy);
            pk[16 + i] = pack2<PT>(f2_lo(left), f2_hi(left));
        }
        chain::tmem_st32(s_tm + 32u * c, pk);
    }
    const uint64_t both = f2_add(sum[0], sum[1]);
    return f2_lo(both) + f2_hi(both);
}

// The same for the open block of a bf16 cache, whose keys have a power of two each (backs: their inverses, in shared memory)
// and whose P has bf16 parts (16 bits), 0 unless `some` -> (sum, m, l, move).  Out of line, because the loop over the full
// blocks must stay small: 1000 rows after 7000 keys took 218 us with this inside the masked step, 196 us beside it, 165 us so.
__device__ __noinline__ float4 soften_open(uint32_t s_tm, int seen, float factor, uint32_t backs, float shift, float m, float l,
                                           bool some) {
    uint32_t r[2][32];
    tmem_ld_32x32b_x32(s_tm, r[0]);
    tmem_ld_32x32b_x32(s_tm + 32u, r[1]);
    tmem_wait_ld(r[0]);
    tie32(r[1]);
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
            float x[4];
            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]) : "r"(backs + 128u * c + 4u * i));
#pragma unroll
            for (int j = 0; j < 4; ++j) r[c][i + j] = __float_as_uint(__uint_as_float(r[c][i + j]) * (x[j] * factor));
        }
    float move = 1.f;
    const float sum = soften<true, __nv_bfloat16>(r, seen, 1.f, shift, m, l, move, s_tm);
    if (!some) {
        tmem_wait_st();
#pragma unroll
        for (int i = 0; i < 32; ++i) r[0][i] = 0;
        chain::tmem_st32(s_tm, r[0]);
        chain::tmem_st32(s_tm + 32u, r[0]);
    }
    return make_float4(sum, m, l, move);
}

// A bounded wait for roles that run ahead: the thread sleeps between its looks.
__device__ __forceinline__ bool warp_wait_idle(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err) {
    int ok = 1;
    if ((threadIdx.x & 31) == 0) ok = mbar_wait_backoff(bar, parity, abort_flag, err, DB_DEV_ERR_TIMEOUT_CVT);
    ok = __shfl_sync(0xffffffffu, ok, 0);
    __syncwarp();
    return ok != 0;
}

template <typename T>
__global__ void __launch_bounds__(THREADS, 1) kv8_rows_kernel(AttnArgs a) {
    constexpr bool WIDE = !std::is_same<T, __half>::value;  // the open block may pass f16's range
    constexpr uint32_t INF = WIDE ? 0x7f80u : 0x7c00u;
    extern __shared__ uint8_t rows_smem[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(rows_smem) + 1023) & ~uintptr_t(1023));
    uint8_t* ring = smem + Q_BYTES;
    Shared& sh = *reinterpret_cast<Shared*>(ring + STAGES * STAGE);
    volatile int* abort_flag = &sh.abort;
    int* err = a.kv.error;
    const int tid = threadIdx.x, lane = tid & 31, warp = chain::warp_index();
    const int h = blockIdx.y, b = blockIdx.z, Hk = a.kv.c.kv_heads;
    pdl_wait();
    pdl_trigger();
    if (blockIdx.x == 0) zero_cut_rows<T>(a, b, h * a.group, a.group);
    int start, count, len;
    item_of(a.kv, b, start, count, len);
    // the last tiles see the most keys: they start first
    const int rows = count * a.group, row0 = (int)(gridDim.x - 1 - blockIdx.x) * ROWS;
    if (row0 >= rows) return;
    const int last = len + (min(row0 + ROWS, rows) - 1) / a.group;  // last key that a row sees
    const int whole = (len + count) / BLK, blocks = last / BLK + 1;
    const int tiles = (blocks + 1) & ~1, pairs = tiles / 2;  // (an odd count is filled up by a tile without keys)
    const int inside = blocks > whole ? len + count - whole * BLK : 0;  // tokens of the open block, where it is read
    const int64_t tail_at = ((int64_t)b * Hk + h) * BLK * D;
    const T* kt = static_cast<const T*>(a.kv.c.k_tail) + tail_at;
    const T* vt = static_cast<const T*>(a.kv.c.v_tail) + tail_at;

    if (tid == 0) {
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(&sh.bars[FULL + i], 1);
            mbar_init(&sh.bars[EMPTY + i], 1);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&sh.bars[S_FULL + i], 1);
            mbar_init(&sh.bars[P_FULL + i], 4);
            mbar_init(&sh.bars[PV_DONE + i], 1);
        }
        mbar_init(&sh.bars[JOIN], 8);
        mbar_init(&sh.bars[MMA_DONE], 1);
        mbar_init(&sh.bars[MMA_DONE + 1], 1);
        mbar_init(&sh.bars[END], THREADS / 32);
        sh.abort = 0;
        sh.tail_v = 0;
        sh.odd = 0;
        fence_barrier_init();
    }
    if (warp == 12) {
        tmem_alloc(&sh.tmem, 512);
        tmem_relinquish();
    }
    // queries to [2^7, 2^8) per row, K-major and 128-byte swizzled: two columns of 64 dims x 128 rows
    const float sign = a.factor < 0.f ? -1.f : 1.f;
    for (int r = warp; r < ROWS; r += THREADS / 32) {
        float x[4] = {0.f, 0.f, 0.f, 0.f};
        const int row = row0 + r;
        if (row < rows) {
            const T* q = static_cast<const T*>(a.q) + (int64_t)(start + row / a.group) * a.ldq +
                         ((int64_t)h * a.group + row % a.group) * D + 4 * lane;
            const uint2 w = *reinterpret_cast<const uint2*>(q);
            x[0] = from_bits<T>(w.x & 0xffffu), x[1] = from_bits<T>(w.x >> 16);
            x[2] = from_bits<T>(w.y & 0xffffu), x[3] = from_bits<T>(w.y >> 16);
        }
        float top = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
        top = warp_max(top);
        float back = 1.f;
        const float up = sign * (top < INFINITY ? code_power(top, back) : 1.f);
        if (lane == 0) sh.row_factor[r] = fabsf(a.factor) * back;
        const uint32_t at = (lane >> 4) * Q_HALF + r * 128 + ((((lane & 15) >> 1) ^ (r & 7)) << 4) + 8 * (lane & 1);
        *reinterpret_cast<uint2*>(smem + at) = make_uint2(pack2<__half>(x[0] * up, x[1] * up), pack2<__half>(x[2] * up, x[3] * up));
    }
    __syncthreads();
    // The open block is exact, whatever its tokens' magnitudes: f16 as it is (its value scale is 1); bf16 keys as f16 after a
    // power of two each, which goes into their scores, and bf16 values as bf16 after one for all, with P's parts in bf16.
    {
        uint32_t vm = 0;
        bool odd = false;
        for (int e = tid; inside && e < BLK * D / 8; e += THREADS) {
            uint32_t km = 0;
            const uint4 k = *reinterpret_cast<const uint4*>(kt + 8 * e), v = *reinterpret_cast<const uint4*>(vt + 8 * e);
            const uint32_t kw[4] = {k.x, k.y, k.z, k.w}, vw[4] = {v.x, v.y, v.z, v.w};
            const bool key_there = e / (D / 8) < inside;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t x = kw[j >> 1] >> (16 * (j & 1)) & 0x7fffu, y = vw[j >> 1] >> (16 * (j & 1)) & 0x7fffu;
                if (key_there && x < INF) km = max(km, x);
                if (8 * e % BLK + j < inside) {
                    if (y < INF) vm = max(vm, y); else odd = true;
                }
            }
            if constexpr (WIDE) {
                // 16 lanes hold a key
#pragma unroll
                for (int o = 8; o; o >>= 1) km = max(km, __shfl_xor_sync(0xffffffffu, km, o));
                if (lane % 16 == 0) sh.key_up[e / 16] = code_power(from_bits<T>(km), sh.key_back[e / 16]);
            }
        }
        if (inside) {
            if constexpr (WIDE) {
                vm = __reduce_max_sync(0xffffffffu, vm);
                if (lane == 0) atomicMax(&sh.tail_v, vm);
            }
            if (__any_sync(0xffffffffu, odd) && lane == 0) sh.odd = 1;
        }
    }
    fence_proxy_async_smem();  // the query tile
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    float vt_back = 1.f;
    const float vt_up = WIDE ? code_power(from_bits<T>(sh.tail_v), vt_back) : 1.f;

    if (warp < 4 || warp > 13) {
        // ---------------------------------------------------------------- codes -> f16 tiles
        // load i, in the order of use: K 0, K 1, then per pair p: K 2p+2, K 2p+3 (while there are), V 2p, V 2p+1
        const int loads = 2 * tiles;
        auto what = [&](int i, bool& is_v) {
            is_v = false;
            if (i < 2) return i;
            int p = (i - 2) >> 2, r = (i - 2) & 3;
            if (p == pairs - 1) r += 2;
            is_v = r >= 2;
            return is_v ? 2 * p + r - 2 : 2 * p + 2 + r;
        };
        // Each warp takes every 6th load whole: what a load costs once (its page, its barriers, the proxy fence) is
        // then paid by six at a time.  A lane holds 16 pieces of 16 codes; a piece's place is refilled with the
        // warp's next load as soon as it is converted.  Page numbers are read one load further ahead.
        const int known = min(blocks, whole);
        auto table = [&](int i) {
            bool is_v;
            const int j = i < loads ? what(i, is_v) : known;
            return j < known && j < a.kv.c.table_width ? a.kv.c.page_table[(int64_t)b * a.kv.c.table_width + j] : -1;
        };
        auto codes_of = [&](int i, int p) -> const uint4* {
            bool is_v;
            if (i < loads) what(i, is_v);
            if (i >= loads || (unsigned)p >= (unsigned)a.kv.c.pages) return nullptr;
            return reinterpret_cast<const uint4*>((is_v ? a.kv.c.v_codes : a.kv.c.k_codes) + ((int64_t)p * Hk + h) * BLK * D);
        };
        // piece c of this lane: 8 lanes that store together take four pieces of one half of two rows (of keys), or of two
        // rows (of values): eight different banks
        auto piece = [&](int c, bool is_v) {
            return is_v ? lane + 32 * c : (4 * c + 2 * (lane >> 4) + ((lane >> 2) & 1)) * 8 + ((lane >> 3) & 1) * 4 + (lane & 3);
        };
        auto first_is_v = [&](int i) {
            bool is_v = false;
            if (i < loads) what(i, is_v);
            return is_v;
        };
        uint4 raw[16];
        const int mine = warp < 4 ? warp : warp - 10;
        int page = table(mine), next_page = table(mine + CONVERTERS);
        float ks = 0.f, vs = 0.f;  // the block's scales, with its codes
        auto scales_of = [&](int i, int p) {
            if (i < loads && !first_is_v(i) && (unsigned)p < (unsigned)a.kv.c.pages) {
                ks = a.kv.c.k_scales[(int64_t)p * Hk + h];
                vs = a.kv.c.v_scales[(int64_t)p * Hk + h];
            }
        };
        {
            const uint4* src = codes_of(mine, page);
            if (src)
#pragma unroll
                for (int c = 0; c < 16; ++c) raw[c] = src[piece(c, first_is_v(mine))];
            scales_of(mine, page);
        }
        for (int i = mine; i < loads; i += CONVERTERS) {
            bool is_v;
            const int j = what(i, is_v), st = i % STAGES;
            const bool tail = j == whole && inside, paged = (unsigned)page < (unsigned)a.kv.c.pages;
            if (j < known && !paged && lane == 0 && err) atomicOr(err, DB_DEV_ERR_SHAPE);
            Info n;
            n.ks = paged ? ks : 1.f;
            const float v_scale = paged ? vs : vt_back;
            scales_of(i + CONVERTERS, next_page);
            const uint4* src = codes_of(i + CONVERTERS, next_page);
            const bool next_v = first_is_v(i + CONVERTERS);
            if (!warp_wait_idle(&sh.bars[EMPTY + st], ((i / STAGES) & 1) ^ 1u, abort_flag, err)) break;
            uint8_t* dst = ring + st * STAGE;
            // rows of 128 bytes: a key's 64 dims, a value feature's 64 tokens; piece 0's row and first half of 16 bytes
            const int q0 = piece(0, is_v), r0 = is_v ? q0 >> 2 : q0 >> 3, half = is_v ? 0 : (q0 >> 2) & 1, p0 = 2 * (q0 & 3);
            const int n0 = piece(0, next_v), step = is_v ? 8 : 4;
#pragma unroll
            for (int c = 0; c < 16; ++c) {
                uint32_t f[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                if (paged) {
                    codes_to_f16(raw[c].x, f[0], f[1]);
                    codes_to_f16(raw[c].y, f[2], f[3]);
                    codes_to_f16(raw[c].z, f[4], f[5]);
                    codes_to_f16(raw[c].w, f[6], f[7]);
                }
                if (src) raw[c] = src[n0 + 32 * c];
                const int r = r0 + step * c;
                uint8_t* row = dst + half * K_HALF + r * 128;
                sts128u(row, (p0 ^ (r & 7)) << 4, f[0], f[1], f[2], f[3]);
                sts128u(row, ((p0 + 1) ^ (r & 7)) << 4, f[4], f[5], f[6], f[7]);
            }
            if (tail) {
#pragma unroll 1
                for (int c = 0; c < 16; ++c) {
                    const int q = piece(c, is_v);
                    const uint4* from = reinterpret_cast<const uint4*>((is_v ? vt : kt) + 16 * q);
                    const uint4 x = from[0], y = from[1];
                    const uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
                    const float up = is_v ? vt_up : WIDE ? sh.key_up[q >> 3] : 1.f;
                    uint32_t f[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        uint32_t l = w[e] & 0xffffu, g = w[e] >> 16;
                        const int key = is_v ? 16 * (q & 3) + 2 * e : q >> 3;
                        // slots without a token, and values (not keys) that are not finite, stay out of the products
                        if (key >= inside || (is_v && (l & INF) == INF)) l = 0;
                        if (key + (is_v ? 1 : 0) >= inside || (is_v && (g & INF) == INF)) g = 0;
                        const float a = from_bits<T>(l) * up, b = from_bits<T>(g) * up;
                        f[e] = !WIDE ? l | g << 16 : is_v ? pack2<T>(a, b) : pack2<__half>(a, b);
                    }
                    const int r = is_v ? q >> 2 : q >> 3, half = is_v ? 0 : (q >> 2) & 1, p0 = 2 * (q & 3);
                    const uint32_t row = half * K_HALF + r * 128;
                    sts128u(dst, row + ((p0 ^ (r & 7)) << 4), f[0], f[1], f[2], f[3]);
                    sts128u(dst, row + (((p0 + 1) ^ (r & 7)) << 4), f[4], f[5], f[6], f[7]);
                }
            }
            if (!is_v && lane == 0) {
                const bool some = v_scale >= FLT_MIN && v_scale < INFINITY;
                const float f = __uint_as_float((__float_as_uint(v_scale) & 0x7fffffu) | 0x3f800000u);
                n.e = some ? (int)(__float_as_uint(v_scale) >> 23) - 127 : NO_SCALE;
                n.lf = some ? log2f(f) : v_scale < FLT_MIN ? 0.f : NAN;
                n.inv = some ? __fdividef(1.f, f) : v_scale < FLT_MIN ? 1.f : NAN;
                n.there = paged || tail;
                sh.info[j & (INFO - 1)] = n;
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.bars[FULL + st]);
            page = next_page;
            next_page = table(i + 2 * CONVERTERS);
        }
    } else if (warp >= 12) {
        // ---------------------------------------------------------------- MMA issue, one parity of tiles
        constexpr uint32_t IDESC_S = idesc_f16_f32(ROWS, BLK), IDESC_O = idesc_f16_f32(ROWS, D);
        constexpr uint32_t IDESC_OPEN = WIDE ? IDESC_O | 1u << 7 | 1u << 10 : IDESC_O;  // (bf16 x bf16)
        const int t = warp - 12;
        const uint64_t dQ = sw128_desc(smem_u32(smem)), dR = sw128_desc(smem_u32(ring));
        const uint32_t s_tm = tmem + 128u * t, o_tm = tmem + TM_O + 128u * t;
        bool ok = true;
        auto loaded = [&](int i) -> int {  // the stage of load i, once it is there
            const int st = i % STAGES;
            ok = ok && warp_wait(&sh.bars[FULL + st], (i / STAGES) & 1, abort_flag, err, DB_DEV_ERR_TIMEOUT_MMA);
            return st;
        };
        // S of pair p goes where the P of pair p - 2 was: after its P V
        auto scores = [&](int p) {
            const int slot = p & 1;
            if (p >= 2) ok = warp_wait(&sh.bars[PV_DONE + 2 * t + slot], ((p >> 1) & 1) ^ 1u, abort_flag, err, DB_DEV_ERR_TIMEOUT_MMA);
            const int st = loaded(p ? 4 * p - 2 + t : t);
            if (!ok) return;
            tc_fence_after();
            if (chain::elect()) {
                const uint64_t dK = dR + (uint64_t)((st * STAGE) >> 4);
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk)
                    umma_f16(s_tm + 64u * slot, dQ + (uint64_t)(((kk >> 2) * Q_HALF + (kk & 3) * 32) >> 4),
                             dK + (uint64_t)(((kk >> 2) * K_HALF + (kk & 3) * 32) >> 4), IDESC_S, kk > 0);
                umma_commit(&sh.bars[EMPTY + st]);
                umma_commit(&sh.bars[S_FULL + 2 * t + slot]);
            }
            __syncwarp();
        };
        auto context = [&](int p) {
            const int slot = p & 1, st = loaded(4 * p + (p == pairs - 1 ? 2 : 4) + t);
            ok = ok && warp_wait(&sh.bars[P_FULL + 2 * t + slot], (p >> 1) & 1, abort_flag, err, DB_DEV_ERR_TIMEOUT_MMA);
            if (!ok) return;
            tc_fence_after();
            // (the descriptor a constant of each branch: an operand that is not keeps the MMAs' others out of uniform registers)
            auto issue = [&](auto idesc) {
                if (chain::elect()) {
                    const uint64_t dV = dR + (uint64_t)((st * STAGE) >> 4);
#pragma unroll
                    for (int kk = 0; kk < BLK / 16; ++kk) {
                        // 32 keys lie in 32 columns: 16 of the first parts, 16 of the second
                        const uint32_t at = s_tm + 64u * slot + 32u * (kk >> 1) + 8u * (kk & 1);
                        chain::umma_f16_ts(o_tm, at + 16u, dV + (uint64_t)(kk * 2), idesc, p > 0 || kk > 0);
                        chain::umma_f16_ts(o_tm, at, dV + (uint64_t)(kk * 2), idesc, 1);
                    }
                    umma_commit(&sh.bars[EMPTY + st]);
                    umma_commit(&sh.bars[PV_DONE + 2 * t + slot]);
                }
            };
            if (WIDE && 2 * p + t == whole && inside)
                issue(std::integral_constant<uint32_t, IDESC_OPEN>());
            else
                issue(std::integral_constant<uint32_t, IDESC_O>());
            __syncwarp();
        };
        scores(0);
        if (pairs > 1 && ok) scores(1);
        for (int p = 0; p < pairs && ok; ++p) {
            context(p);
            if (p + 2 < pairs && ok) scores(p + 2);
        }
        // every MMA issued has completed before tensor memory is released
        if (chain::elect()) {
            umma_commit(&sh.bars[MMA_DONE + t]);
            mbar_wait_drain(&sh.bars[MMA_DONE + t], 0, DRAIN_NS);
        }
        __syncwarp();
    } else {
        // ---------------------------------------------------------------- softmax
        const int t = (warp - 4) >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t o_tm = tmem + lanes + TM_O + 128u * t;
        const int limit = row0 + row < rows ? len + (row0 + row) / a.group : -1;
        const float factor = sh.row_factor[row];
        float m = -INFINITY, l = 0.f;
        int unit = NO_SCALE, largest = NO_SCALE;  // O is in units of 2^(unit - SHIFT)
        bool ok = true;
        for (int p = 0; p < pairs; ++p) {
            const int slot = p & 1, base = (2 * p + t) * BLK;
            const uint32_t s_tm = tmem + lanes + 128u * t + 64u * slot;
            if (!(ok = warp_wait(&sh.bars[S_FULL + 2 * t + slot], (p >> 1) & 1, abort_flag, err, DB_DEV_ERR_TIMEOUT_EPI))) break;
            tc_fence_after();
            const Info n = sh.info[(2 * p + t) & (INFO - 1)];
            const int seen = n.there ? limit - base : -1;  // keys 0 .. seen of the tile
            float move = 1.f, all;
            int raise = 0;
            if (n.there && n.e != NO_SCALE) {
                if (unit == NO_SCALE) {
                    unit = n.e + 2;  // (O is 0 so far)
                } else if (n.e >= unit || n.e < unit - 6) {
                    const int next = max(n.e + 2, largest - 80);
                    raise = unit - next;
                    unit = next;
                }
                largest = max(largest, unit);
            }
            const int down = n.e == NO_SCALE ? LEAST : max(SHIFT + n.e - unit, LEAST);
            const float shift = (float)down + n.lf;
            uint32_t r[2][32];
            if (WIDE && 2 * p + t == whole && inside) {
                const float4 x = soften_open(s_tm, seen, factor, smem_u32(sh.key_back), shift, m, l, down > LEAST);
                all = x.x, m = x.y, l = x.z, move = x.w;
            } else {
                tmem_ld_32x32b_x32(s_tm, r[0]);
                tmem_ld_32x32b_x32(s_tm + 32u, r[1]);
                tmem_wait_ld(r[0]);
                tie32(r[1]);
                const float scale = factor * n.ks;
                if (__any_sync(0xffffffffu, seen < BLK - 1))
                    all = soften<true>(r, seen, scale, shift, m, l, move, s_tm);
                else
                    all = soften<false>(r, seen, scale, shift, m, l, move, s_tm);
            }
            if (all != 0.f) l = fmaf(all, n.inv * power2(-down), l);
            move *= power2(raise);
            // O is stable once the previous P V of this parity is done
            const bool rescale = p > 0 && __any_sync(0xffffffffu, move != 1.f);
            if (rescale) {
                if (!(ok = warp_wait(&sh.bars[PV_DONE + 2 * t + (slot ^ 1)], ((p - 1) >> 1) & 1, abort_flag, err, DB_DEV_ERR_TIMEOUT_EPI))) break;
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    tmem_ld_32x32b_x32(o_tm + 32u * c, r[0]);
                    tmem_wait_ld(r[0]);
#pragma unroll
                    for (int i = 0; i < 32; ++i) r[0][i] = __float_as_uint(__uint_as_float(r[0][i]) * move);
                    chain::tmem_st32(o_tm + 32u * c, r[0]);
                }
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.bars[P_FULL + 2 * t + slot]);
        }
        // the last P V of both parities, then the two halves together: this warpgroup writes 64 features
        for (int x = 0; x < 2 && ok; ++x)
            ok = warp_wait(&sh.bars[PV_DONE + 2 * x + ((pairs - 1) & 1)], ((pairs - 1) >> 1) & 1, abort_flag, err, DB_DEV_ERR_TIMEOUT_EPI);
        if (ok) {
            tc_fence_after();
            sh.join_m[t][row] = m;
            sh.join_l[t][row] = l;
            sh.join_unit[t][row] = unit;
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.bars[JOIN]);
            ok = warp_wait(&sh.bars[JOIN], 0, abort_flag, err, DB_DEV_ERR_TIMEOUT_EPI);
        }
        if (ok) {
            const float m0 = sh.join_m[0][row], m1 = sh.join_m[1][row], mm = fmaxf(m0, m1), at = mm == -INFINITY ? 0.f : mm;
            const float f0 = ex2(m0 - at), f1 = ex2(m1 - at), sum = sh.join_l[0][row] * f0 + sh.join_l[1][row] * f1;
            const int u0 = sh.join_unit[0][row], u1 = sh.join_unit[1][row], u = max(u0, u1);
            const float norm = sum == 0.f ? 0.f : 1.f / sum, back = ldexpf(1.f, u - SHIFT);  // no key could be read: 0
            const float g0 = f0 * power2(u0 - u) * norm, g1 = f1 * power2(u1 - u) * norm;
            const int n = row0 + row;
            T* out = static_cast<T*>(a.out) + (int64_t)(start + n / a.group) * a.ldo + ((int64_t)h * a.group + n % a.group) * D + 64 * t;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t e[32], o[32];
                const uint32_t from = tmem + lanes + TM_O + 64u * t + 32u * c;
                tmem_ld_32x32b_x32(from, e);
                tmem_ld_32x32b_x32(from + 128u, o);
                tmem_wait_ld(e);
                tie32(o);
                float v[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = (__uint_as_float(e[i]) * g0 + __uint_as_float(o[i]) * g1) * back;
                if (sh.odd) {
                    // values of the open block that are not finite reach the rows that see their tokens
                    for (int key = 0; key < min(inside, limit - whole * BLK + 1); ++key)
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const float x = to_f32(vt[(64 * t + 32 * c + i) * BLK + key]);
                            if (!isfinite(x)) v[i] += x;
                        }
                }
                if (n < rows) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        *reinterpret_cast<uint4*>(out + 32 * c + 8 * i) =
                            make_uint4(pack2<T>(v[8 * i], v[8 * i + 1]), pack2<T>(v[8 * i + 2], v[8 * i + 3]),
                                       pack2<T>(v[8 * i + 4], v[8 * i + 5]), pack2<T>(v[8 * i + 6], v[8 * i + 7]));
                }
            }
        }
    }
    // through an mbarrier: every role is done with tensor memory before it is released
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.bars[END]);
    if (warp == 12) {
        if (lane == 0) mbar_wait_drain(&sh.bars[END], 0, DB_WAIT_LIMIT_NS);
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

}  // namespace

template <typename T>
cudaError_t kv8_rows_attention(const AttnArgs& a, cudaStream_t stream) {
    const cudaError_t e = db_set_max_smem(reinterpret_cast<const void*>(kv8_rows_kernel<T>), SMEM);
    if (e != cudaSuccess) return e;
    const int64_t tiles = ((int64_t)a.kv.max_rows * a.group + ROWS - 1) / ROWS;
    return db_launch_pdl(kv8_rows_kernel<T>, dim3((unsigned)tiles, a.kv.c.kv_heads, a.kv.items), dim3(THREADS), SMEM, stream, a);
}
template cudaError_t kv8_rows_attention<__half>(const AttnArgs&, cudaStream_t);
template cudaError_t kv8_rows_attention<__nv_bfloat16>(const AttnArgs&, cudaStream_t);

}  // namespace db
