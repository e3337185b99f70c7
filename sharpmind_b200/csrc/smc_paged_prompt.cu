// Attention of many rows over the paged cache (a prompt, a chunk of one, long drafts) on the fifth-generation tensor cores.
//
// One CTA = up to 256 (row, query head) pairs of one sequence and KV head, two tiles of 128, a thread a pair; keys in steps of 64.  The codes are brought as
// they lie in their pages, turned to fp16 (exact) by four warps and stored as 128-byte-swizzled K-major tiles, once for all heads of a group and both
// tiles.  Scores S = Q K^T and outputs O += P V are tcgen05.mma, fp16 with fp32 sums in tensor memory, P in the columns that S leaves:
//   bfloat16  queries exact in fp16 after a power of two per row, weights rounded to 11 bits
//   fp32      queries and weights as hi + lo, two products each: 22 bits, of weights as long as they are 2^-3 or more (lo, too, goes in steps of 2^-24)
// With the pages' scales, constant over 16 keys:  y = S f + b, f = s_k * row factor, b = log2(s_v);  w = 2^(y - R);  l = sum w / s_v;  out = O / l.
// R is 6 below the maximum of y of a row's first step and goes up (to 6 below the maximum) only where a step's weights sum up to more than fp16 holds: a step takes
// no maximum, and O, in tensor memory, is rarely multiplied again.  What is left below a weight's last step, 2^-25 at most, is lost to O: 2^-31 of the largest of the first step, in
// both types (a first key that takes all but 2^-20 of the weight and has no value leaves the others 11 bits each).  The sum l loses nothing: its weights are fp32.
// Warp roles:  0 .. 3, 4 .. 7  softmax of tile 0, 1      8 .. 11  codes to fp16      12, 13  MMA issue of tile 0, 1
// Scores have two buffers a tile, so a softmax finds its next ones there.
// Few pairs: the steps are split over CTAs, whose partial results a second kernel joins.
// Measured (6000 bf16 rows, 32 query heads, 8 of keys, of 128): 394 us, 748 TFLOP/s, 44 % of a bf16 matmul's rate; 1.46 us a step.  With 3000 rows the tensor pipe is active 30 % of the time and issue
// slots 41 %: the chain from scores to weights bounds it, no unit.  Leaving out the exponentials gained 1 %, all MMAs 7 %, the stores of the converted tiles 11 %.
#include "smc_paged.cuh"
#include "smc_tc.cuh"

namespace {

constexpr int PAIRS = 256, TILE = 128, KT = 64, G = KT / 16, SOFT_WARPS = 8, CONV_WARP = 8, MMA_WARP = 12, THREADS = 32 * (MMA_WARP + 2), SC_SLOTS = 8, STEPS_LEAST = 4;
constexpr float R_BELOW = 6.0f, SUM_MOST = 65000.0f;
// A step with a value scale 2^SCALES_NEAR or more below an earlier one takes a pass of its own for the softmax's sum, over 2^(R - SUM_UP).  (Under nearer scales a key that
// w loses is 2^-68 of a larger one.  The pass is the step's own loop once more: in code of its own it cost every step, 6000 rows 407 us; so, as without it, 392 to 394.)
constexpr int SCALES_NEAR = 64;
constexpr float SUM_UP = 48.0f, SUM_DOWN = 0x1p-48f;

// A wait names a phase by its parity: no barrier passes a phase before its waiter has seen the one before.  (PV_DONE may for a softmax, which looks
// at it only in step i for the product of step i - 1, where neither the one before can be missing nor the one after be there.)
enum { FULL = 0, EMPTY = 4, S_FULL = 8, P_FULL = 12 /* [tile][step parity] */, PV_DONE = 16, Q_FULL = 18, O_FULL = 20, BARS = 22 };

template <int HD, bool SPLIT>
struct Shape {
    static constexpr int PLANES = SPLIT ? 2 : 1, STAGES = 2;  // (each stage has its own copy of the MMAs: four took 398 us where two take 392, 6000 rows)
    static constexpr uint32_t SUB_Q = TILE * 128, Q_PLANE = HD / 64 * SUB_Q, Q_TILE = PLANES * Q_PLANE;
    static constexpr uint32_t HALF = KT * HD * 2, STAGE = 2 * HALF;  // fp16 keys of a step, values of the last step but one
    static constexpr uint32_t OFF_K = 2 * Q_TILE, OFF_SC = OFF_K + STAGES * STAGE, OFF_BAR = OFF_SC + SC_SLOTS * G * 16, SMEM = OFF_BAR + 256;
    static constexpr uint32_t COL_S = 0, COL_O = 4 * KT, COLS = 512;  // scores [tile][step parity]
    static_assert(BARS * 8 + 8 <= 256 && SMEM <= 227 * 1024 && COL_O + 2 * HD <= COLS && STAGES + 2 < SC_SLOTS, "");
};
// tcgen05.mma whose operands are known at compile time, up to the shared memory's base: operands that come through registers take an issuing
// thread some 140 clocks an MMA (measured here), these less than the MMA itself.  D, A_COL: columns of tensor memory, all of which is the CTA's, so it starts
// at 0; A, B: byte offsets of swizzled tiles; base: low word of the descriptor of offset 0.
constexpr uint32_t DESC_HIGH = (1024u >> 4) | (1u << 14) | (2u << 29);
template <uint32_t D, uint32_t A, uint32_t B, uint32_t IDESC>
__device__ __forceinline__ void mma_ss(uint32_t base, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b32 a, b, d, i;\n\t.reg .b64 x, y;\n\tadd.u32 a, %0, %2;\n\tadd.u32 b, %0, %3;\n\tmov.b64 x, {a, %6};\n\tmov.b64 y, {b, %6};\n\t"
        "mov.u32 d, %4;\n\tmov.u32 i, %5;\n\tsetp.ne.b32 p, %1, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [d], x, y, i, p;\n\t}" ::"r"(base),
        "r"(accumulate), "n"(A >> 4), "n"(B >> 4), "n"(D), "n"(IDESC), "n"(DESC_HIGH)
        : "memory");
}
template <uint32_t D, uint32_t A_COL, uint32_t B, uint32_t IDESC>
__device__ __forceinline__ void mma_ts(uint32_t base, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b32 a, b, d, i;\n\t.reg .b64 y;\n\tadd.u32 b, %0, %3;\n\tmov.b64 y, {b, %6};\n\tmov.u32 a, %2;\n\t"
        "mov.u32 d, %4;\n\tmov.u32 i, %5;\n\tsetp.ne.b32 p, %1, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [d], [a], y, i, p;\n\t}" ::"r"(base),
        "r"(accumulate), "n"(A_COL), "n"(B >> 4), "n"(D), "n"(IDESC), "n"(DESC_HIGH)
        : "memory");
}
// f(integral constants 0 .. N - 1)
template <int I> struct ic {
    static constexpr int v = I;
};
template <int N, int I = 0, class F>
__device__ __forceinline__ void each(F &&f)
{
    if constexpr (I < N) {
        f(ic<I>());
        each<N, I + 1>(f);
    }
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t *r)
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
        "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]),
                 "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w)
{
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ uint32_t half2_bits(float a, float b)
{
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t rest_bits(float a, float b, uint32_t hi)
{
    const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
    return half2_bits(a - h.x, b - h.y);
}
// two fp32 operations an instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
// power of two that brings a row's largest magnitude to [2^14, 2^15)
__device__ __forceinline__ int row_shift(float most) { return min(14 - ((int)(__float_as_uint(most) >> 23) - 127), 126); }
__host__ __device__ constexpr uint32_t idesc_f16(int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(TILE >> 4) << 24); }

// One thread issues a tile's MMAs: at step x, O += P(x - 2) V(x - 2) and the scores of x.  These take the columns that P(x - 2) is in.  Only MMAs of one accumulator
// and shape are promised to run in their order, so the scores wait until the product has completed; the softmax of x - 1 runs meanwhile.
template <int HD, bool SPLIT, int TILE_NO>
__device__ __forceinline__ void issue_mmas(uint32_t sbase, int mine, int n, uint32_t bars, volatile uint32_t *abort_flag, int *status)
{
    using S = Shape<HD, SPLIT>;
    static_assert(S::STAGES % 2 == 0, "");
    const uint32_t base = ((sbase >> 4) & 0x3FFFu) | (1u << 16);
    auto bar = [&](int i) { return bars + 8u * (uint32_t)i; };
    auto wait = [&](int i, uint32_t parity) { smc_tc_wait(bar(i), parity & 1u, abort_flag, status); };
    bool there = false;  // the next stage, as far as is known
    auto step = [&](auto stage, int x) {  // x % STAGES = stage
        constexpr int st = decltype(stage)::v, next = (st + 1) % S::STAGES;
        if (!there) wait(FULL + st, (uint32_t)(x / S::STAGES));
        if (x >= 2 && x - 2 < mine) wait(P_FULL + 2 * TILE_NO + st % 2, (uint32_t)((x - 2) >> 1));
        smc_tc_fence_after();
        there = smc_mbar_test(bar(FULL + next), (uint32_t)((x + 1) / S::STAGES) & 1u);
        if (x >= 2 && x - 2 < mine) {
            each<S::PLANES * (KT / 16)>([&](auto i) {
                constexpr int p = S::PLANES - 1 - decltype(i)::v / (KT / 16), kk = decltype(i)::v % (KT / 16);  // smallest products first
                mma_ts<S::COL_O + TILE_NO * HD, S::COL_S + (2 * TILE_NO + st % 2) * KT + p * (KT / 2) + kk * 8, S::OFF_K + st * S::STAGE + S::HALF + kk * 32, idesc_f16(HD)>(
                    base, decltype(i)::v > 0 || x > 2);
            });
            smc_tc_commit(bar(PV_DONE + TILE_NO));
            if (x - 1 == mine) smc_tc_commit(bar(O_FULL + TILE_NO));
        }
        if (x < mine) {
            if (x >= 2) {
                wait(PV_DONE + TILE_NO, (uint32_t)(x - 2));
                smc_tc_fence_after();
            }
            each<S::PLANES * (HD / 16)>([&](auto i) {
                constexpr int p = S::PLANES - 1 - decltype(i)::v / (HD / 16), ks = decltype(i)::v % (HD / 16);
                mma_ss<S::COL_S + (2 * TILE_NO + st % 2) * KT, TILE_NO * S::Q_TILE + p * S::Q_PLANE + ks / 4 * S::SUB_Q + ks % 4 * 32,
                       S::OFF_K + st * S::STAGE + ks / 4 * (KT * 128) + ks % 4 * 32, idesc_f16(KT)>(base, decltype(i)::v > 0);
            });
            smc_tc_commit(bar(S_FULL + 2 * TILE_NO + st % 2));
        }
        if (x < mine + 2 && mine > 0) smc_tc_commit(bar(EMPTY + st));
        else smc_mbar_arrive(bar(EMPTY + st));  // the other tile goes on
    };
    if (mine > 0) wait(Q_FULL + TILE_NO, 0u);
#pragma unroll 1
    for (int x0 = 0; x0 < n + 2; x0 += S::STAGES)
        each<S::STAGES>([&](auto i) {
            if (x0 + decltype(i)::v < n + 2) step(i, x0 + decltype(i)::v);
        });
}

// Row and head within the group of every step-th pair, divided once
struct PairWalk {
    int row, head, group, rows, heads;
    __device__ __forceinline__ PairWalk(int pair, int group_, int step) : row(pair / group_), group(group_), rows(step / group_)
    {
        head = pair - row * group, heads = step - rows * group;
    }
    __device__ __forceinline__ void next()
    {
        row += rows, head += heads;
        if (head >= group) head -= group, ++row;
    }
};
// What a CTA does: pairs [m0, m0 + pairs) of sequence s and head h; key tiles [kv0, kv0 + n[t]) of tile t, of which this piece takes [i0, i1).
struct Job {
    int s, h, m0, pairs, len, n_rows, r0, from, kv0, n0, n1, i0, i1, piece, pieces;
};
__device__ __forceinline__ bool job_of(const smc_paged_view &c, const smc_paged_query &u, int item, int h, int piece, int split, Job &j, int *status)
{
    const int group = u.heads / c.kvh;
    auto items_before = [&](int s) { return (int)((long long)min(max(c.row_start ? c.row_start[s] : s, 0), c.rows) * group / PAIRS) + s; };
    int lo = 0, hi = c.batch;  // the last sequence whose items start at or before this one
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (items_before(mid) <= item) lo = mid;
        else hi = mid;
    }
    const smc_paged_seq sq = smc_paged_sequence(c, lo);
    if ((sq.bad || sq.n > u.max_rows) && status) *status = SMC_STATUS_PAGED;
    const int local = item - items_before(lo);
    const long long all = (long long)sq.n * group;
    if (local < 0 || (long long)local * PAIRS >= all) return false;
    j.s = lo, j.h = h, j.m0 = local * PAIRS, j.pairs = (int)min((long long)PAIRS, all - j.m0);
    j.len = sq.len, j.n_rows = sq.n, j.r0 = sq.r0;
    const int p0 = sq.len - sq.n;  // position of the sequence's first row
    const int first = p0 + j.m0 / group, end0 = p0 + (j.m0 + min(j.pairs, TILE) - 1) / group + 1, end1 = p0 + (j.m0 + j.pairs - 1) / group + 1;
    j.from = u.window > 0 ? max(0, first - u.window + 1) : 0;
    j.kv0 = j.from / KT;
    j.n0 = max(1, (end0 + KT - 1) / KT - j.kv0), j.n1 = j.pairs > TILE ? max(j.n0, (end1 + KT - 1) / KT - j.kv0) : j.n0;
    j.pieces = min(split, max(1, j.n1 / (u.bf16 ? STEPS_LEAST : 2 * STEPS_LEAST))), j.piece = piece;
    if (piece >= j.pieces) return false;
    j.i0 = (int)((long long)piece * j.n1 / j.pieces), j.i1 = (int)((long long)(piece + 1) * j.n1 / j.pieces);
    return true;
}

template <typename T, int HD>
__global__ void __launch_bounds__(THREADS, 1) paged_prompt_kernel(const smc_paged_view c, const smc_paged_query u, int items, int split, float *work, int *status)
{
    constexpr bool SPLIT = sizeof(T) == 4;
    using S = Shape<HD, SPLIT>;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t sbase = smc_smem_u32(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile uint32_t *abort_flag = reinterpret_cast<volatile uint32_t *>(smem + S::OFF_BAR + BARS * 8 + 4);
    auto bar = [&](int i) { return sbase + S::OFF_BAR + 8u * (uint32_t)i; };
    auto wait = [&](int i, uint32_t parity) {  // by whole warps
        smc_tc_wait(bar(i), parity & 1u, abort_flag, status);
        __syncwarp();
    };
    auto arrive = [&](int i) {
        __syncwarp();
        if (lane == 0) smc_mbar_arrive(bar(i));
    };
    // tensor memory is taken after the predecessor has completed and before the successor may start
    asm volatile("griddepcontrol.wait;" ::: "memory");
    Job j;
    {
        int b = blockIdx.x;
        const int piece = b % split;
        b /= split;
        const int h = b % c.kvh, item = items - 1 - b / c.kvh;  // later rows see more keys: they start first
        if (!job_of(c, u, item, h, piece, split, j, threadIdx.x == 0 ? status : nullptr)) {  // (the same for all threads)
            asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
            return;
        }
    }
    if (threadIdx.x == 0) {
        const uint32_t readers = j.pairs > TILE ? 2u : 1u;
        for (int i = 0; i < S::STAGES; ++i) smc_mbar_init(bar(FULL + i), 4), smc_mbar_init(bar(EMPTY + i), readers);
        for (int i = 0; i < 4; ++i) smc_mbar_init(bar(S_FULL + i), 1), smc_mbar_init(bar(P_FULL + i), 4);
        for (int i = 0; i < 2; ++i) smc_mbar_init(bar(PV_DONE + i), 1), smc_mbar_init(bar(O_FULL + i), 1), smc_mbar_init(bar(Q_FULL + i), 4);
        *abort_flag = 0;
        smc_fence_barrier_init();
    }
    if (warp == MMA_WARP) {
        __syncwarp();
        smc_tc_alloc(sbase + S::OFF_BAR + BARS * 8, S::COLS);
    }
    smc_tc_fence_before();
    __syncthreads();
    smc_tc_fence_after();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(smem + S::OFF_BAR + BARS * 8);
    const int group = u.heads / c.kvh;
    const bool two = j.pairs > TILE;
    const int stop0 = min(j.n0, j.i1), stop1 = two ? j.i1 : j.i0;  // tile t takes [i0, stop)

    if (warp < SOFT_WARPS) {
        const int t = warp >> 2, rl = 32 * (warp & 3) + lane, m = t * TILE + rl, stop = t ? stop1 : stop0;
        const bool real = m < j.pairs;
        const int pair = j.m0 + (real ? m : 0), tok = pair / group;
        const uint32_t lanes = tmem + ((uint32_t)(32 * (warp & 3)) << 16), col_s0 = lanes + S::COL_S + (uint32_t)(2 * t * KT), col_o = lanes + S::COL_O + (uint32_t)(t * HD);
        const int pos = j.len - j.n_rows + tok;
        // 16 bytes of the warp's own rows in its tile's queries
        auto own = [&](int row, int chunk) {
            const int block = chunk >> 3;
            return sbase + (uint32_t)t * S::Q_TILE + (uint32_t)(block / (HD / 64)) * S::Q_PLANE + (uint32_t)(block % (HD / 64)) * S::SUB_Q + (uint32_t)(32 * (warp & 3) + row) * 128u +
                   (uint32_t)(((chunk & 7) ^ (row & 7)) << 4);
        };
        float rowf = 0.0f, R = -INFINITY, l = 0.0f;
        if (stop > j.i0) {
            // the warp's 32 rows, 16 bytes a lane, the lanes of a row side by side; a short loop, four of a lane's loads ahead: code that is
            // gone through once a CTA costs its fetch
            constexpr int N = 16 / (int)sizeof(T), LANES = HD / N, AT_ONCE = 32 / LANES;
            const int e = lane % LANES * N, sub = lane / LANES;
            float mine = 0.0f;  // the largest magnitude of this lane's own row
            constexpr int AHEAD = 4;
            PairWalk from(j.m0 + t * TILE + 32 * (warp & 3) + sub, group, AT_ONCE);
            const T *const q0 = static_cast<const T *>(u.q) + (long long)j.r0 * u.q_stride + (size_t)(j.h * group) * HD + e;
            uint4 next[AHEAD];
            auto fetch = [&](int r0) {
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) {
                    const bool in = r0 < 32 && t * TILE + 32 * (warp & 3) + r0 + i * AT_ONCE + sub < j.pairs;
                    next[i] = in ? *reinterpret_cast<const uint4 *>(q0 + (long long)from.row * u.q_stride + (size_t)from.head * HD) : make_uint4(0, 0, 0, 0);
                    from.next();
                }
            };
            fetch(0);
#pragma unroll 1
            for (int r0 = 0; r0 < 32; r0 += AHEAD * AT_ONCE) {
              uint4 raw[AHEAD];
#pragma unroll
              for (int i = 0; i < AHEAD; ++i) raw[i] = next[i];
              fetch(r0 + AHEAD * AT_ONCE);
              float tops[AHEAD];
#pragma unroll
              for (int i = 0; i < AHEAD; ++i) {
                tops[i] = 0.0f;
#pragma unroll
                for (int k = 0; k < N; ++k) tops[i] = fmaxf(tops[i], fabsf(to_f(reinterpret_cast<const T *>(&raw[i])[k])));
              }
#pragma unroll
              for (int o = LANES / 2; o > 0; o >>= 1)
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) tops[i] = fmaxf(tops[i], __shfl_xor_sync(0xFFFFFFFFu, tops[i], o));
#pragma unroll
              for (int i = 0; i < AHEAD; ++i) {
                const int r = r0 + i * AT_ONCE, row = 32 * (warp & 3) + r + sub;
                const float most = tops[i], theirs = __shfl_sync(0xFFFFFFFFu, most, (lane % AT_ONCE) * LANES);
                if (lane / AT_ONCE * AT_ONCE == r) mine = theirs;
                float v[N];
#pragma unroll
                for (int k = 0; k < N; ++k) v[k] = to_f(reinterpret_cast<const T *>(&raw[i])[k]);
                // the largest magnitude of the row goes to [2^14, 2^15); a negative scale turns the queries' sign
                float fac = __uint_as_float((uint32_t)(row_shift(most) + 127) << 23);
                if (u.scale < 0.0f) fac = -fac;
                uint32_t hi[N / 2], lo[N / 2];
#pragma unroll
                for (int k = 0; k < N / 2; ++k) {
                    hi[k] = half2_bits(v[2 * k] * fac, v[2 * k + 1] * fac);
                    if (SPLIT) lo[k] = rest_bits(v[2 * k] * fac, v[2 * k + 1] * fac, hi[k]);
                }
                const uint32_t dst = own(row & 31, e >> 3);
                if constexpr (SPLIT) {
                    const uint32_t half = (uint32_t)(e & 4) * 2u;
                    smc_sts64(dst + half, make_uint2(hi[0], hi[1])), smc_sts64(dst + S::Q_PLANE + half, make_uint2(lo[0], lo[1]));
                } else {
                    sts128(dst, hi[0], hi[1], hi[2], hi[3]);
                }
              }
            }
            rowf = fabsf(u.scale) * 1.44269504088896341f * __uint_as_float((uint32_t)(127 - row_shift(mine)) << 23);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            arrive(Q_FULL + t);
        }
        // rows of this tile: [lowest, highest] positions, for tiles that every row sees whole
        const int lowest = j.len - j.n_rows + (j.m0 + t * TILE) / group, highest = j.len - j.n_rows + (j.m0 + min(j.pairs, (t + 1) * TILE) - 1) / group;
        bool there = false;  // the next scores, as far as is known
#pragma unroll 1
        for (int i = j.i0; i < stop; ++i) {
            const int it = i - j.i0, key0 = (j.kv0 + i) * KT;
            const uint32_t col_s = col_s0 + (uint32_t)((it & 1) * KT);
            if (!__all_sync(0xFFFFFFFFu, there)) wait(S_FULL + 2 * t + (it & 1), (uint32_t)(it >> 1));
            smc_tc_fence_after();
            uint32_t s[KT];
#pragma unroll
            for (int k = 0; k < KT; k += 16) smc_tc_ld16(col_s + (uint32_t)k, *reinterpret_cast<uint32_t(*)[16]>(s + k));
            float4 x[G];
            const float4 *sc = reinterpret_cast<const float4 *>(smem + S::OFF_SC) + (it % SC_SLOTS) * G;
#pragma unroll
            for (int k = 0; k < G; ++k) x[k] = sc[k];
            smc_tc_wait_ld();
            const bool inner = key0 + KT <= lowest + 1 && (u.window <= 0 || key0 > highest - u.window);
            const int hi = inner ? KT : pos - key0, lo = !inner && u.window > 0 ? hi - u.window : -1;  // keys lo + 1 .. hi of the tile are seen
            if (!inner) {
#pragma unroll
                for (int k = 0; k < KT; ++k)
                    if (k > hi) s[k] = 0xFF800000u;  // -infinity
                if (lo >= 0) {
#pragma unroll
                    for (int k = 0; k < KT; ++k)
                        if (k <= lo) s[k] = 0xFF800000u;
                }
            }
            // scales of 16 keys, for this row: a factor above 0, so that hidden keys stay -infinity; nothing of keys that are all hidden
#pragma unroll
            for (int k = 0; k < G; ++k) {
                x[k].x = fmaxf(x[k].x * rowf, 1e-37f);
                if (!inner && (16 * k > hi || 16 * k + 15 <= lo)) x[k].y = -INFINITY, x[k].z = 0.0f;
            }
            float add, far = x[0].w;
#pragma unroll 1
            for (bool again = true;;) {
                const float ref = R == -INFINITY ? 0.0f : R;
                float total = 0.0f;
                add = 0.0f;
#pragma unroll
                for (int k = 0; k < G; ++k) {
                    const float2 f = make_float2(x[k].x, x[k].x), bias = make_float2(x[k].y - ref, x[k].y - ref);
                    float2 w[8];
                    uint32_t p[8], rest[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        w[e] = fma2(make_float2(__uint_as_float(s[16 * k + 2 * e]), __uint_as_float(s[16 * k + 2 * e + 1])), f, bias);
                        w[e].x = ex2(w[e].x), w[e].y = ex2(w[e].y);
                        p[e] = half2_bits(w[e].x, w[e].y);
                        if constexpr (SPLIT) rest[e] = rest_bits(w[e].x, w[e].y, p[e]);
                    }
                    tmem_st8(col_s + (uint32_t)(8 * k), p);
                    if constexpr (SPLIT) tmem_st8(col_s + (uint32_t)(KT / 2 + 8 * k), rest);
                    const float2 sum2 = add2(add2(add2(w[0], w[1]), add2(w[2], w[3])), add2(add2(w[4], w[5]), add2(w[6], w[7])));
                    const float sum = sum2.x + sum2.y;
                    total += sum, add = fmaf(sum, x[k].z, add);
                }
                // No maximum is taken where the weights' sum tells that none of them is too large.  (A row's first step has no R yet.)
                const bool bad = again && (R == -INFINITY || total > SUM_MOST);
                if (!__any_sync(0xFFFFFFFFu, bad || far != 0.0f)) break;
                if (!__any_sync(0xFFFFFFFFu, bad)) {
                    if (far == 1.0f) {  // R is this step's from here: a pass for the sum alone
                        far = 2.0f, again = false;
#pragma unroll
                        for (int k = 0; k < G; ++k) x[k].y = x[k].y == -INFINITY ? x[k].y : SUM_UP;
                    } else {  // and the weights once more, which add nothing to it
                        l = fmaf(total, SUM_DOWN, l), far = 0.0f;
#pragma unroll
                        for (int k = 0; k < G; ++k) x[k].y = x[k].y == -INFINITY ? x[k].y : sc[k].y, x[k].z = 0.0f;
                    }
                    tmem_wait_st();
                    continue;
                }
                again = false;
                tmem_wait_st();
                float top = -INFINITY;
#pragma unroll
                for (int k = 0; k < G; ++k) {
                    float m4[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        m4[e] = fmaxf(fmaxf(__uint_as_float(s[16 * k + e]), __uint_as_float(s[16 * k + 4 + e])), fmaxf(__uint_as_float(s[16 * k + 8 + e]), __uint_as_float(s[16 * k + 12 + e])));
                    top = fmaxf(top, fmaf(fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])), x[k].x, x[k].y));  // (what is not a number a maximum drops)
                }
                float down = 0.0f;
                if (bad && top > -INFINITY) {
                    const float was = R;
                    R = top - R_BELOW;
                    down = was - R;
                }
                const float corr = ex2(down);
                l = smc_paged_fold(l, down, 0.0f);
                if (it > 0) {
                    wait(PV_DONE + t, (uint32_t)(it - 1));  // (the one before that: these scores waited for it)
                    smc_tc_fence_after();
#pragma unroll 1
                    for (int k = 0; k < HD; k += 16) {
                        uint32_t o[16];
                        smc_tc_ld16(col_o + (uint32_t)k, o);
                        smc_tc_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                        tmem_st16(col_o + (uint32_t)k, o);
                    }
                }
            }
            l += add;
            there = i + 1 < stop && smc_mbar_test(bar(S_FULL + 2 * t + ((it + 1) & 1)), (uint32_t)((it + 1) >> 1) & 1u);  // (the answer comes under what follows)
            tmem_wait_st();
            smc_tc_fence_before();
            arrive(P_FULL + 2 * t + (it & 1));
        }
        if (stop > j.i0) {
            wait(O_FULL + t, 0u);
            smc_tc_fence_after();
            const float norm = l == 0.0f ? 0.0f : 1.0f / l;
            // Rows leave through the queries' shared memory, which no product reads any more: a lane its own row first, then 16 bytes a lane with the lanes of a
            // row side by side.  Results, or what a piece has of O, half a row (fp32: a row) at a time.
            constexpr int N = 16 / (int)sizeof(T), AT_ONCE = S::PLANES * HD / 2;
            const bool piece = j.pieces > 1;
            float *part = work + ((size_t)blockIdx.x * PAIRS) * (HD + 4);
#pragma unroll 1
            for (int k0 = 0; k0 < HD; k0 += AT_ONCE) {
                uint32_t o[AT_ONCE];
#pragma unroll
                for (int k = 0; k < AT_ONCE; k += 16) smc_tc_ld16(col_o + (uint32_t)(k0 + k), *reinterpret_cast<uint32_t(*)[16]>(o + k));
                smc_tc_wait_ld();
                if (piece || SPLIT) {
                    const float by = piece ? 1.0f : norm;
#pragma unroll
                    for (int e = 0; e < AT_ONCE; e += 4)
                        sts128(own(lane, e / 4), __float_as_uint(__uint_as_float(o[e]) * by), __float_as_uint(__uint_as_float(o[e + 1]) * by),
                               __float_as_uint(__uint_as_float(o[e + 2]) * by), __float_as_uint(__uint_as_float(o[e + 3]) * by));
                } else {
#pragma unroll
                    for (int e = 0; e < AT_ONCE; e += 8)
                        sts128(own(lane, e / 8), pack2(__uint_as_float(o[e]) * norm, __uint_as_float(o[e + 1]) * norm), pack2(__uint_as_float(o[e + 2]) * norm, __uint_as_float(o[e + 3]) * norm),
                               pack2(__uint_as_float(o[e + 4]) * norm, __uint_as_float(o[e + 5]) * norm), pack2(__uint_as_float(o[e + 6]) * norm, __uint_as_float(o[e + 7]) * norm));
                }
                __syncwarp();
                if (piece) {
                    constexpr int CHUNKS = AT_ONCE / 4;
#pragma unroll 2
                    for (int r = lane / CHUNKS, c = lane % CHUNKS; r < 32; r += 32 / CHUNKS) {
                        const int at = t * TILE + 32 * (warp & 3) + r;
                        if (at < j.pairs) *reinterpret_cast<uint4 *>(part + (size_t)at * (HD + 4) + k0 + 4 * c) = smc_lds128(own(r, c));
                    }
                } else {
                    constexpr int CHUNKS = AT_ONCE / N;
                    PairWalk to(j.m0 + t * TILE + 32 * (warp & 3) + lane / CHUNKS, group, 32 / CHUNKS);
                    T *const out0 = static_cast<T *>(u.out) + ((size_t)j.r0 * u.heads + j.h * group) * HD + k0 + lane % CHUNKS * N;
#pragma unroll 2
                    for (int r = lane / CHUNKS; r < 32; r += 32 / CHUNKS, to.next())
                        if (t * TILE + 32 * (warp & 3) + r < j.pairs)
                            *reinterpret_cast<uint4 *>(out0 + ((size_t)to.row * u.heads + to.head) * HD) = smc_lds128(own(r, lane % CHUNKS));
                }
                __syncwarp();
            }
            if (piece && real) part[(size_t)m * (HD + 4) + HD] = R, part[(size_t)m * (HD + 4) + HD + 1] = l;
        } else if (real && j.pieces > 1) {  // a piece behind the last key that this tile sees
            float *part = work + ((size_t)blockIdx.x * PAIRS + m) * (HD + 4);
            const float zero[4] = {};
            for (int k = 0; k < HD; k += 4) smc_paged_store4(part + k, zero);
            part[HD] = -INFINITY, part[HD + 1] = 0.0f;
        }
    } else if (warp < MMA_WARP) {
        // ---------------------------------------------------------------- codes to fp16
        const int w = warp - CONV_WARP, page = 1 << c.shift, r8 = lane & 7, q4 = lane >> 3;
        constexpr int UNITS = KT * HD / 16 / 128;  // of 16 codes a thread: 8 keys x 64 dims, 8 dims x 64 keys a warp
        constexpr int IN_K = HD / 64, IN_V = KT / 64, STEP_K = 4 / IN_K, STEP_V = 4 / IN_V;
        // unit x of this warp: keys 8 (w / IN_K + STEP_K x) .., dims 64 (w % IN_K) + 16 q4 ..; dims 8 (w / IN_V + STEP_V x) .., keys 64 (w % IN_V) + 16 q4 ..
        const int hi = min(j.len, j.len - j.n_rows + (j.m0 + j.pairs - 1) / group + 1);  // keys [from, hi) count
        const uint32_t stride = (uint32_t)(c.kvh * HD) << c.shift;                         // bytes of a page
        const uint8_t *k_base = c.k + ((size_t)j.h * HD << c.shift) + 64 * (w % IN_K) + 16 * q4, *v_base = c.v + ((size_t)j.h * HD << c.shift) + ((size_t)(8 * (w / IN_V) + r8) << c.shift);
        const int v_group = 4 * (w % IN_V) + q4;
        const uint32_t swizzle = (uint32_t)(r8 * 128 + ((2 * q4) ^ r8) * 16), flip = (uint32_t)((2 * q4 ^ r8) * 16) ^ (uint32_t)(((2 * q4 + 1) ^ r8) * 16);
        const uint32_t k_dst = sbase + S::OFF_K + (uint32_t)((w % IN_K) * KT * 128 + w / IN_K * 1024), v_dst = sbase + S::OFF_K + S::HALF + (uint32_t)((w % IN_V) * HD * 128 + w / IN_V * 1024);
        // Page of this lane's group of 16 keys (lane % G) of tile i, or -1.  Codes of page 0 stand in for those of a page that is not there: nothing of a
        // key that no row sees reaches a result, and undefined codes among the values are made zeros below.
        auto page_of = [&](int i) {
            const int key = (j.kv0 + i) * KT + 16 * (lane % G), p0 = key >> c.shift << c.shift;
            if (i >= j.i1 || p0 + page <= j.from || p0 >= hi) return -1;  // (pages that left the window may have gone to another sequence)
            const int id = smc_paged_page(c, j.s, key >> c.shift);
            if (id < 0) *status = SMC_STATUS_PAGED;
            return id;
        };
        auto scales_of = [&](int id) { return id < 0 ? make_float2(0.0f, 0.0f) : *reinterpret_cast<const float2 *>(c.scales + 2 * ((size_t)id * c.kvh + j.h)); };
        auto fetch_k = [&](int ids, int x) {
            const int in_tile = 8 * (w / IN_K + STEP_K * x), id = max(__shfl_sync(0xFFFFFFFFu, ids, in_tile >> 4), 0);
            return __ldcg(reinterpret_cast<const uint4 *>(k_base + (size_t)(uint32_t)id * stride + ((in_tile & (page - 1)) + r8) * HD));
        };
        auto fetch_v = [&](const uint8_t *v_page, int x) { return __ldcg(reinterpret_cast<const uint4 *>(v_page + ((8 * STEP_V * x) << c.shift))); };
        auto place = [&](uint32_t at, const uint4 &v) {
            const uint32_t raw[4] = {v.x, v.y, v.z, v.w};
            uint32_t h[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) h[2 * e] = smc_e4m3x2_half2(raw[e] & 0xFFFFu), h[2 * e + 1] = smc_e4m3x2_half2(raw[e] >> 16);
            sts128(at, h[0], h[1], h[2], h[3]);
            sts128(at ^ flip, h[4], h[5], h[6], h[7]);
        };
        // step x brings the keys of x and the values of x - 2; codes of the next step of each are on their way meanwhile
        const int n = j.i1 - j.i0;
        uint4 raw_k[UNITS], raw_v[UNITS];
        int id_k = page_of(j.i0), id_1 = -1, id_v = -1;  // pages of the keys of step x, of those before, of the values
        float2 sc = scales_of(id_k);
        int largest = -127;  // log2 of the largest value scale so far
#pragma unroll
        for (int i = 0; i < UNITS; ++i) raw_k[i] = fetch_k(id_k, i);
#pragma unroll 1
        for (int x = 0; x < n + 2; ++x) {
            const int st = x % S::STAGES, id_next = page_of(j.i0 + x + 1);
            wait(EMPTY + st, (uint32_t)(x / S::STAGES) ^ 1u);  // (a fresh barrier passes the first)
            if (x >= 2) {
                const int key0 = (j.kv0 + j.i0 + x - 2) * KT;
                if (key0 < j.from || key0 + KT > hi || __any_sync(0xFFFFFFFFu, id_v < 0)) {  // values of keys that do not count are zeros
                    const int v_id = __shfl_sync(0xFFFFFFFFu, id_v, v_group);
                    uint32_t keep[4] = {};
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int key = key0 + 16 * v_group + e;
                        if (v_id >= 0 && key >= j.from && key < hi) keep[e >> 2] |= 0xFFu << (8 * (e & 3));
                    }
#pragma unroll
                    for (int i = 0; i < UNITS; ++i) raw_v[i].x &= keep[0], raw_v[i].y &= keep[1], raw_v[i].z &= keep[2], raw_v[i].w &= keep[3];
                }
#pragma unroll
                for (int i = 0; i < UNITS; ++i) place(v_dst + (uint32_t)st * S::STAGE + (uint32_t)(STEP_V * i) * 1024u + swizzle, raw_v[i]);
            }
            id_v = id_1, id_1 = id_k;
            const uint8_t *v_page = v_base + (size_t)(uint32_t)max(__shfl_sync(0xFFFFFFFFu, id_v, v_group), 0) * stride + ((16 * v_group) & (page - 1));
#pragma unroll
            for (int i = 0; i < UNITS; ++i) raw_v[i] = fetch_v(v_page, i);
            if (x < n) {
                if (w == 0) {  // (its lanes have the step's groups of keys, again and again)
                    // scale of keys; log2 and reciprocal of that of values (a power of two's exponent); 1 where the step's value scales lie far below an earlier one.
                    // An undefined one of either makes the second undefined
                    const int log2v = id_k < 0 ? -127 : smc_paged_log2(sc.y);
                    largest = max(largest, __reduce_max_sync(0xFFFFFFFFu, log2v));
                    const float both = sc.x + sc.y, e = (float)log2v, far = __any_sync(0xFFFFFFFFu, id_k >= 0 && log2v < largest - SCALES_NEAR) ? 1.0f : 0.0f;
                    if (lane < G)
                        reinterpret_cast<float4 *>(smem + S::OFF_SC)[(x % SC_SLOTS) * G + lane] =
                            id_k < 0 ? make_float4(0.0f, -INFINITY, 0.0f, far) : make_float4(sc.x, both == both ? e : both, 1.0f / sc.y, far);
                }
#pragma unroll
                for (int i = 0; i < UNITS; ++i) place(k_dst + (uint32_t)st * S::STAGE + (uint32_t)(STEP_K * i) * 1024u + swizzle, raw_k[i]);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            arrive(FULL + st);
            id_k = id_next;
            sc = scales_of(id_k);
#pragma unroll
            for (int i = 0; i < UNITS; ++i) raw_k[i] = fetch_k(id_k, i);
        }
    } else if (lane == 0) {
        // ---------------------------------------------------------------- MMA issue
        const int n = j.i1 - j.i0;
        if (warp == MMA_WARP) issue_mmas<HD, SPLIT, 0>(sbase, stop0 - j.i0, n, bar(0), abort_flag, status);
        else if (two) issue_mmas<HD, SPLIT, 1>(sbase, stop1 - j.i0, n, bar(0), abort_flag, status);
    }
    __syncwarp();
    smc_tc_fence_before();
    __syncthreads();
    if (warp == MMA_WARP) {
        __syncwarp();
        smc_tc_dealloc(tmem, S::COLS);
    }
}

// One warp = JOIN_WARP pairs of a job whose keys were split: joins the pieces in their order.  Latency and L2 bound it: drafts' 576 blocks 7.4 us, three prompts' 1024 19 (cold caches).
template <typename T, int HD, int JOIN_WARP>
__global__ void __launch_bounds__(256) paged_prompt_join_kernel(const smc_paged_view c, const smc_paged_query u, int items, int split, const float *__restrict__ work)
{
    smc_grid_dep_sync();
    constexpr int E = HD / 32, JOIN_PAIRS = 8 * JOIN_WARP;
    const int lane = threadIdx.x & 31, b = blockIdx.x / (PAIRS / JOIN_PAIRS), m0 = blockIdx.x % (PAIRS / JOIN_PAIRS) * JOIN_PAIRS + (threadIdx.x >> 5) * JOIN_WARP;
    Job j;
    if (!job_of(c, u, items - 1 - b / c.kvh, b % c.kvh, 0, split, j, nullptr) || j.pieces == 1 || m0 >= j.pairs) return;
    const size_t step = (size_t)PAIRS * (HD + 4);
    const int group = u.heads / c.kvh;
    const float *row[JOIN_WARP];
    float2 end[JOIN_WARP];  // a lane a piece: R and l
    float o[JOIN_WARP][E] = {};
#pragma unroll
    for (int k = 0; k < JOIN_WARP; ++k) {
        row[k] = work + ((size_t)b * split * PAIRS + min(m0 + k, j.pairs - 1)) * (HD + 4);
        end[k] = lane < j.pieces ? *reinterpret_cast<const float2 *>(row[k] + lane * step + HD) : make_float2(-INFINITY, 0.0f);
    }
    float f[JOIN_WARP], sum[JOIN_WARP];
#pragma unroll
    for (int k = 0; k < JOIN_WARP; ++k) {
        float top = end[k].x;
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
        const float down = end[k].x - (top == -INFINITY ? 0.0f : top);
        f[k] = ex2(down);
        sum[k] = smc_group_sum<32>(lane < j.pieces ? smc_paged_fold(end[k].y, down, 0.0f) : 0.0f);
    }
#pragma unroll 2
    for (int i = 0; i < j.pieces; ++i)
#pragma unroll
        for (int k = 0; k < JOIN_WARP; ++k) {
            const float w = __shfl_sync(0xFFFFFFFFu, f[k], i);
#pragma unroll
            for (int e = 0; e < E; ++e) o[k][e] = fmaf(row[k][i * step + lane + 32 * e], w, o[k][e]);
        }
#pragma unroll
    for (int k = 0; k < JOIN_WARP; ++k) {
        const int pair = j.m0 + m0 + k, tok = pair / group;
        if (m0 + k >= j.pairs) break;
        T *dst = static_cast<T *>(u.out) + ((size_t)(j.r0 + tok) * u.heads + j.h * group + pair - tok * group) * HD;
#pragma unroll
        for (int e = 0; e < E; ++e) dst[lane + 32 * e] = from_f<T>(sum[k] == 0.0f ? 0.0f : o[k][e] / sum[k]);
    }
}

// Jobs of a call (some may be empty: a sequence's share is rounded up), and into how many pieces each one's keys go: as many as the device takes at once for one
// sequence, whose pieces are alike in length (512 bf16 rows behind 5000 keys: 81 us, twice as many 89; 1000 rows 123 / 146; 700 rows the other way, 118 / 110), and
// twice as many for several of their own lengths (three: 124 us, as many as at once 142, four times as many 142).  A piece has four steps at least (drafts, 8 x 35
// pairs over 2000 keys: 17.5 us, two 19.9, eight 21.2), in fp32, whose queries are longer in coming, eight.
long long items_of(int batch, int rows, int group) { return (long long)rows * group / PAIRS + batch; }
int split_of(const smc_ctx *ctx, int kvh, int batch, int rows, int group, int max_len)
{
    const long long jobs = items_of(batch, rows, group) * kvh;
    return (int)std::max(1LL, std::min({(long long)max_len / KT / STEPS_LEAST, (batch == 1 ? 1LL : 2LL) * ctx->sm_count / std::max(1LL, jobs), 32LL}));  // (a lane a piece joins them)
}

}  // namespace

size_t smc_paged_prompt_work(const smc_ctx *ctx, int kvh, int batch, int rows, int heads, int hd, int max_len)
{
    const int split = split_of(ctx, kvh, batch, rows, heads / kvh, max_len);
    return split == 1 ? 0 : (size_t)items_of(batch, rows, heads / kvh) * kvh * split * PAIRS * (hd + 4) * sizeof(float);
}

int smc_launch_paged_prompt(smc_ctx *ctx, const smc_paged_view &c, const smc_paged_query &u, float *work, cudaStream_t s)
{
    const int group = u.heads / c.kvh, split = split_of(ctx, c.kvh, c.batch, c.rows, group, u.max_len);
    const long long items = items_of(c.batch, c.rows, group);
    if (items * c.kvh * split * (PAIRS / 8) > 0x7FFFFFFF || (long long)c.rows * group > 0x7FFFFFFF)
        return smc_fail(ctx, SMC_E_UNSUPPORTED, "paged_attention: %d rows of %d sequences in one call", c.rows, c.batch);
    const long long jobs = items * c.kvh;
    auto go = [&](auto main, auto few, auto many, uint32_t smem) {
        cudaFuncSetAttribute(main, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        smc_launch_dep(ctx->use_pdl, main, dim3((unsigned)(jobs * split)), dim3(THREADS), smem, s, c, u, (int)items, split, work, ctx->d_status);
        if (split == 1) return;
        // (a warp a pair while the device takes them all at once, four else: drafts 17.5 us, the other way 22.1; three prompts 123.5, 126.1)
        if (jobs * (PAIRS / 8) <= 8LL * ctx->sm_count) smc_launch_dep(ctx->use_pdl, few, dim3((unsigned)(jobs * (PAIRS / 8))), dim3(256), 0, s, c, u, (int)items, split, work);
        else smc_launch_dep(ctx->use_pdl, many, dim3((unsigned)(jobs * (PAIRS / 32))), dim3(256), 0, s, c, u, (int)items, split, work);
    };
    if (u.bf16)
        u.hd == 128 ? go(paged_prompt_kernel<bf16, 128>, paged_prompt_join_kernel<bf16, 128, 1>, paged_prompt_join_kernel<bf16, 128, 4>, Shape<128, false>::SMEM)
                    : go(paged_prompt_kernel<bf16, 64>, paged_prompt_join_kernel<bf16, 64, 1>, paged_prompt_join_kernel<bf16, 64, 4>, Shape<64, false>::SMEM);
    else
        u.hd == 128 ? go(paged_prompt_kernel<float, 128>, paged_prompt_join_kernel<float, 128, 1>, paged_prompt_join_kernel<float, 128, 4>, Shape<128, true>::SMEM)
                    : go(paged_prompt_kernel<float, 64>, paged_prompt_join_kernel<float, 64, 1>, paged_prompt_join_kernel<float, 64, 4>, Shape<64, true>::SMEM);
    SMC_LAUNCH_CHECK(ctx);
    return SMC_OK;
}
