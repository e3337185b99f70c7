// Attention of a few rows of every sequence over the paged cache (a decode step, drafts): the whole cache passes once through registers, so HBM is
// the bound, and the work has to be even over the device whatever the sequences' lengths are.
//
// Units of 64 keys of one sequence and KV head, in the order (sequence, head, tile); the grid's CTAs take equal runs of them, a CTA's four
// warps take its units in turn.  What a CTA has of one sequence and head (a segment) is merged in shared memory at its end; a segment that a run's
// border cuts leaves as (running maximum, sum, unnormalised output), and a second small kernel joins those.  The order of all sums is fixed by the call's sizes and the lengths.
// More than sixteen pairs are segments of sixteen each, one behind the other, so that the next ones find the keys in L2.
// Measured (bf16, 64 sequences of up to 8000 keys, 583 MB): 122 us with the join, 4.8 TB/s; 192 sequences of one length 5.7.  Some 12 us are fixed: planning, the first copies, join.
// Leaving out the MMAs, the conversions or the exponentials of a copy of it gained nothing.
//
// A warp's unit: keys and values arrive by bulk copies in a ring of its own, K or V of 64 tokens a slot, two slots ahead.  Scores and outputs
// are mma.sync m16n8k16 in fp16 with fp32 sums, transposed: S^T = K Q^T and O^T = V^T P^T, so that the eight columns are the (row, query head) pairs, of which
// there are few, and no tile is half empty.  An e4m3 code is exact in fp16; the queries are scaled by a power of two per row to 2^15 at most, which bfloat16
// ones take exactly; fp32 queries and weights go in as hi + lo, 22 bits (weights as long as they are 2^-3 or more, 2^-17 of the largest), into the same sums.
// Both products' contraction indices are permuted so that a thread reads 16 contiguous codes: thread t of a quad takes dims [16 t, 16 t + 16) (and + 64) of
// the keys, tokens [16 t, 16 t + 16) of the values.  The scores' row i of tile pair M is token 16 (i / 2) + 2 M + i % 2: a transposed eight by eight
// block of weights (movmatrix) then is the second product's operand, and all tokens of a thread's scores lie in one page, so a unit's scales are two numbers.
//   y_j = x_j log2(e) + log2(s_v);  w_j = 2^(y_j - M), M the running maximum of y less 14;  O = sum w_j code_j;  l = sum w_j / s_v;  out = O / l
// The value scales ride in the exponent, so the weights stay within fp16: 2^14 at most, in steps of 2^-24 at least (fp32: hi and lo together), 2^-38 of the largest.
// The sum takes every key whatever the scales are: a thread whose keys' weights all lie below 2^-60, 0 as fp16 numbers, takes them 2^64 up (scales are 2^-40 .. 2^120, so a
// weight may be 2^-150 and count).  That and the sums' way to a new M are worth 0.1 to 0.6 us of a step of single tokens, 4 of 151 for 4 rows over 64 sequences of up to 8000.
#include "smc_async.cuh"
#include "smc_paged.cuh"

namespace {

constexpr int RUNS_MOST = 1024, PART = 16, PARTS_MOST = 4, PART_TILES = 15;
constexpr int WARPS = 4, THREADS = 32 * WARPS, UNIT = 64, SLOTS = 3, CHUNKS = 256;
constexpr float W_SHIFT = 14.0f, W_UP = 64.0f, W_DOWN = 0x1p-64f, LOW = -60.0f;

template <int HD>
struct Ring {
    static constexpr int SLOT = UNIT * HD + 128;               // values of 16- and 32-token pages lie 32 and 64 bytes further apart: no bank conflicts
    static constexpr int OFF_MERGE = WARPS * SLOTS * SLOT;      // [warp][8 rows] of half of O, maximum and sum
    static constexpr int MERGE_ROW = HD / 2 + 4;
    static constexpr int OFF_BAR = OFF_MERGE + WARPS * 8 * MERGE_ROW * 4, OFF_PLAN = OFF_BAR + WARPS * SLOTS * 8;
    static constexpr int SMEM = OFF_PLAN + (CHUNKS + WARPS) * 4 + 16;
};

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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

// an 8 x 8 matrix of halves, two of a row a thread, transposed
__device__ __forceinline__ uint32_t transposed(uint32_t v)
{
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// tiles [t0, t0 + tiles) of 64 keys that rows of sequence s see; one tile, all masked, where there is no key, none where there is no row
struct Span {
    int r0, n, len, from, t0, tiles, parts;  // parts: its pairs in sixteens
    bool bad;
};
template <bool PARTED> __device__ __forceinline__ Span span_of(const smc_paged_view &c, const smc_paged_query &u, int s)
{
    const smc_paged_seq sq = smc_paged_sequence(c, s);
    Span p;
    p.r0 = sq.r0, p.n = min(sq.n, u.max_rows), p.len = sq.len, p.bad = sq.bad || sq.n > u.max_rows;
    p.from = u.window > 0 ? max(0, sq.len - p.n + 1 - u.window) : 0;
    p.t0 = p.from / UNIT;
    p.tiles = p.n == 0 ? 0 : max(1, (sq.len + UNIT - 1) / UNIT - p.t0);
    p.parts = PARTED ? (p.n * (u.heads / c.kvh) + PART - 1) / PART : 1;
    return p;
}
// run of units of CTA i of n: [first, first of the next)
__device__ __forceinline__ int run_first(int i, int n, int units) { return (int)((long long)i * units / n); }
__device__ __forceinline__ int run_of(int unit, int n, int units) { return (int)(((long long)(unit + 1) * n - 1) / units); }

// units of a sequence: those of a head's parts follow one another, so that the next part finds the keys in L2
template <bool PARTED> __device__ __forceinline__ int units_of(const smc_paged_view &c, const Span &p) { return (PARTED ? c.kvh * p.parts : c.kvh) * p.tiles; }
// Where a warp is among the units: sequence s has [base, base + units_of)
struct Place {
    int s, base;
    Span p;
};
template <bool PARTED> __device__ __forceinline__ void advance(const smc_paged_view &c, const smc_paged_query &u, Place &w, int unit)
{
    while (w.base + units_of<PARTED>(c, w.p) <= unit && w.s + 1 < c.batch) {
        w.base += units_of<PARTED>(c, w.p);
        w.p = span_of<PARTED>(c, u, ++w.s);
    }
}

// slot of a CTA's cut segment: 0 where it began before the run, 1 where it begins in it
__device__ __forceinline__ float *partial(float *work, int cta, int which, int rows, int hd) { return work + ((size_t)cta * 2 + which) * rows * (hd + 4); }

// NQ: (row, query head) pairs in eights; PARTED: segments of sixteen pairs each, as many as a sequence's rows need
template <typename T, int HD, int NQ, bool PARTED>
__global__ void __launch_bounds__(THREADS, 2) paged_decode_kernel(const smc_paged_view c, const smc_paged_query u, float *work, int aligned, int *status)
{
    constexpr bool SPLIT = sizeof(T) == 4;  // queries and weights as hi + lo
    constexpr int KS = HD / 16, CH = HD / 64, PL = SPLIT ? 2 : 1;
    using R = Ring<HD>;
    extern __shared__ __align__(128) uint8_t smem[];
    const uint32_t sbase = smc_smem_u32(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int group = u.heads / c.kvh;
    const uint32_t ring = sbase + (uint32_t)(warp * SLOTS * R::SLOT), bars = sbase + (uint32_t)(R::OFF_BAR + warp * SLOTS * 8);
    float *merge = reinterpret_cast<float *>(smem + R::OFF_MERGE);
    int *plan = reinterpret_cast<int *>(smem + R::OFF_PLAN), *sums = plan + CHUNKS;
    if (lane == 0) {
        for (int i = 0; i < SLOTS; ++i) smc_mbar_init(bars + 8 * i, 1);
        smc_fence_barrier_init();
    }
    smc_grid_dep_sync();

    // how many units there are before each of 256 groups of sequences
    const int per = (c.batch + CHUNKS - 1) / CHUNKS;
    int mine[2], local = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        int n = 0;
        for (int s = (2 * (int)threadIdx.x + i) * per, e = min(c.batch, s + per); s < e; ++s) {
            const Span p = span_of<PARTED>(c, u, s);
            n += units_of<PARTED>(c, p);
            if (p.bad && blockIdx.x == 0) *status = SMC_STATUS_PAGED;
        }
        mine[i] = n, local += n;
    }
    int scan = local;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xFFFFFFFFu, scan, o);
        if (lane >= o) scan += v;
    }
    if (lane == 31) sums[warp] = scan;
    __syncthreads();
    int before = scan - local, units = 0;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
        if (i < warp) before += sums[i];
        units += sums[i];
    }
    plan[2 * threadIdx.x] = before, plan[2 * threadIdx.x + 1] = before + mine[0];
    __syncthreads();
    int first, last;
    if (aligned) {  // whole segments
        auto unit_of = [&](long long segment) {
            const int s1 = (int)(segment / c.kvh), g0 = s1 / per;
            if (s1 >= c.batch) return units;
            int before = plan[g0];
            for (int s = g0 * per; s < s1; ++s) before += units_of<PARTED>(c, span_of<PARTED>(c, u, s));
            return before + (int)(segment - (long long)s1 * c.kvh) * (units_of<PARTED>(c, span_of<PARTED>(c, u, s1)) / c.kvh);
        };
        const long long segments = (long long)c.batch * c.kvh;
        first = unit_of(blockIdx.x * segments / gridDim.x), last = unit_of((blockIdx.x + 1) * segments / gridDim.x);
        if (first >= last) return;
    } else {
        const int runs = min((int)gridDim.x, units);  // (no run between two others is empty)
        if ((int)blockIdx.x >= runs) return;
        first = run_first(blockIdx.x, runs, units), last = run_first(blockIdx.x + 1, runs, units);
    }
    Place at;
    {
        int lo = 0, hi = CHUNKS;  // the last group that starts at or before `first`
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (plan[mid] <= first) lo = mid;
            else hi = mid;
        }
        // (groups behind the last sequence start at `units`)
        at.s = min(lo * per, c.batch - 1), at.base = plan[lo], at.p = span_of<PARTED>(c, u, at.s);
        advance<PARTED>(c, u, at, first);
    }

    // ---- what is on its way: half-stages K, V of this warp's units first + warp, + 4, ...
    const int page = 1 << c.shift, pad = c.shift == 4 ? 32 : c.shift == 5 ? 64 : 0, g16 = g >> 1;
    struct Fetch {
        int tile0, h, id, lo, hi;  // the unit's first key, its head, the page of tokens [16 g16, 16 g16 + 16) (-1: nothing to bring); keys that count
    };
    Place ahead = at;
    auto look = [&](int unit) {
        Fetch f{0, 0, -1, 0, 0};
        if (unit >= last) return f;
        advance<PARTED>(c, u, ahead, unit);
        const int rest = unit - ahead.base, hp = rest / ahead.p.tiles;
        f.h = PARTED ? hp / ahead.p.parts : hp, f.tile0 = (ahead.p.t0 + rest - hp * ahead.p.tiles) * UNIT;
        f.lo = ahead.p.from, f.hi = ahead.p.len;
        const int key = f.tile0 + 16 * g16, p0 = key >> c.shift << c.shift;
        if (p0 + page > f.lo && p0 < f.hi) {  // (pages that left the window may have gone to another sequence)
            f.id = smc_paged_page(c, ahead.s, key >> c.shift);
            if (f.id < 0) *status = SMC_STATUS_PAGED;
        }
        return f;
    };
    auto scales_of = [&](const Fetch &f) {
        return f.id < 0 ? make_float2(0.0f, 1.0f) : *reinterpret_cast<const float2 *>(c.scales + 2 * ((size_t)f.id * c.kvh + f.h));
    };
    const bool leader = (lane & 7) == 0 && ((16 * g16) & (page - 1)) == 0;
    auto request = [&](const Fetch &f, bool values, int slot) {
        const bool bring = leader && f.id >= 0;
        const unsigned who = __ballot_sync(0xFFFFFFFFu, bring);
        if (lane == 0) smc_mbar_expect_tx(bars + 8 * slot, (uint32_t)(__popc(who) * page * HD));
        __syncwarp();
        if (bring) {
            const size_t block = ((size_t)f.id * c.kvh + f.h) * ((size_t)HD << c.shift);
            const uint32_t dst = ring + (uint32_t)(slot * R::SLOT + 16 * g16 * HD + (values ? ((16 * g16) >> c.shift) * pad : 0));
            smc_bulk_g2s(dst, (values ? c.v : c.k) + block, (uint32_t)(page * HD), bars + 8 * slot);
        }
    };
    auto landed = [&](int half) {
        if (!smc_mbar_wait(bars + 8 * (half % SLOTS), (uint32_t)(half / SLOTS) & 1u)) *status = 4;
    };
    int unit = first + warp, half = 0;
    Fetch now = look(unit), next = look(unit + WARPS), later;
    float2 sc_now = scales_of(now), sc_next;
    request(now, false, 0), request(now, true, 1), request(next, false, 2);

    // ---- segments
    for (int seg = first; seg < last;) {
        advance<PARTED>(c, u, at, seg);
        const Span p = at.p;
        const int hp = (seg - at.base) / p.tiles, begin = at.base + hp * p.tiles, end = begin + p.tiles, stop = min(end, last);
        const int h = PARTED ? hp / p.parts : hp, m0 = PARTED ? (hp - h * p.parts) * PART : 0, all_pairs = p.n * group, pairs = PARTED ? min(PART, all_pairs - m0) : all_pairs;
        uint32_t q[NQ][PL][KS][2];
        float rowf[NQ][2];  // of rows 2 t, 2 t + 1 of an eight, like all that follows
        int pos[NQ][2];
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) {
            const int m = min(m0 + 8 * nq + g, all_pairs - 1), i = m / group;  // (rows behind the last repeat it and are not stored)
            const T *src = static_cast<const T *>(u.q) + (long long)(p.r0 + i) * u.q_stride + (size_t)(h * group + m - i * group) * HD + 16 * t;
            float x[4 * KS], most = 0.0f;
#pragma unroll
            for (int e = 0; e < KS; ++e) {  // dims 64 (e / 4) + 16 t + 4 (e % 4)
                smc_paged_load4(src + 64 * (e >> 2) + 4 * (e & 3), *reinterpret_cast<float(*)[4]>(x + 4 * e));
#pragma unroll
                for (int j = 0; j < 4; ++j) most = fmaxf(most, fabsf(x[4 * e + j]));
            }
            most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 1));
            most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 2));
            // the largest magnitude goes to [2^14, 2^15)
            const int up = min(14 - ((int)(__float_as_uint(most) >> 23) - 127), 126);
            const float fac = __uint_as_float((uint32_t)(up + 127) << 23), back = u.scale * 1.44269504088896341f * __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
            for (int e = 0; e < 2 * KS; ++e) {
                const float a = x[2 * e] * fac, b = x[2 * e + 1] * fac;
                q[nq][0][e >> 1][e & 1] = half2_bits(a, b);
                if constexpr (SPLIT) q[nq][1][e >> 1][e & 1] = rest_bits(a, b, q[nq][0][e >> 1][e & 1]);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                rowf[nq][e] = __shfl_sync(0xFFFFFFFFu, back, 4 * (2 * t + e));
                pos[nq][e] = p.len - p.n + min(m0 + 8 * nq + 2 * t + e, all_pairs - 1) / group;
            }
        }
        float o[NQ][KS][4] = {}, M[NQ][2], l[NQ][2];
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) M[nq][0] = M[nq][1] = -INFINITY, l[nq][0] = l[nq][1] = 0.0f;

        for (; unit < stop; unit += WARPS) {
            const int key0 = now.tile0 + 16 * g16 + (g & 1);  // this thread's tokens of the scores: key0 + 2 M
            later = look(unit + 2 * WARPS);
            sc_next = scales_of(next);
            // (a power of two's exponent; a scale that is none, left where no page is or undefined, stays what it is)
            const float bias = sc_now.y == sc_now.y ? (float)smc_paged_log2(sc_now.y) : sc_now.y, inv = 1.0f / sc_now.y;
            const bool inner = now.tile0 >= now.lo && now.tile0 + UNIT <= p.len - p.n + 1 && (u.window <= 0 || now.tile0 > p.len - 1 - u.window);
            landed(half);
            float s[NQ][4][4] = {};
            {
                const uint32_t row = ring + (uint32_t)((half % SLOTS) * R::SLOT + (16 * g16 + (g & 1)) * HD + 16 * t);
#pragma unroll
                for (int mt = 0; mt < 4; ++mt)
#pragma unroll
                    for (int ch = 0; ch < CH; ++ch) {
                        const uint4 ra = smc_lds128(row + (uint32_t)(4 * mt * HD + 64 * ch)), rb = smc_lds128(row + (uint32_t)((4 * mt + 2) * HD + 64 * ch));
                        const uint32_t wa[4] = {ra.x, ra.y, ra.z, ra.w}, wb[4] = {rb.x, rb.y, rb.z, rb.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t a[4] = {smc_e4m3x2_half2(wa[e] & 0xFFFFu), smc_e4m3x2_half2(wb[e] & 0xFFFFu), smc_e4m3x2_half2(wa[e] >> 16), smc_e4m3x2_half2(wb[e] >> 16)};
#pragma unroll
                            for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
                                for (int pl = PL - 1; pl >= 0; --pl) mma_f16(s[nq][mt], a, q[nq][pl][4 * ch + e][0], q[nq][pl][4 * ch + e][1]);
                        }
                    }
            }
            __syncwarp();
            request(next, true, half % SLOTS);
            ++half;
            uint32_t w[NQ][PL][8];  // weights as B fragments: block M of tokens
#pragma unroll
            for (int nq = 0; nq < NQ; ++nq) {
                float down[2], add[2];
                uint32_t seen = 0;  // ones where a row's weights are not 2^W_UP up
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float f = rowf[nq][r] * sc_now.x;
#pragma unroll
                    for (int j = 0; j < 8; ++j) s[nq][j >> 1][2 * (j & 1) + r] = fmaf(s[nq][j >> 1][2 * (j & 1) + r], f, bias);
                    if (!inner) {
                        const int hi = min(pos[nq][r], p.len - 1), lo = u.window > 0 ? pos[nq][r] - u.window : -1;
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            if (key0 + 2 * j > hi || key0 + 2 * j <= lo) s[nq][j >> 1][2 * (j & 1) + r] = -INFINITY;
                    }
                    float top = s[nq][0][r];
#pragma unroll
                    for (int j = 1; j < 8; ++j) top = fmaxf(top, s[nq][j >> 1][2 * (j & 1) + r]);
                    const float mine = top;
                    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 4));
                    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 8));
                    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 16));
                    const float nm = fmaxf(M[nq][r], top - W_SHIFT), ref = nm == -INFINITY ? 0.0f : nm;
                    down[r] = M[nq][r] - ref;  // (-inf: nothing yet)
                    M[nq][r] = nm;
                    const bool low = mine - ref < LOW;
                    const float from = low ? ref - W_UP : ref;
                    seen |= low ? 0u : 0xFFFFu << (16 * r);
                    float sum = 0.0f;
#pragma unroll
                    for (int j = 0; j < 8; ++j) sum += s[nq][j >> 1][2 * (j & 1) + r] = ex2(s[nq][j >> 1][2 * (j & 1) + r] - from);
                    // (first by the scale's inverse: neither product leaves fp32.  A row that sees none of these tokens takes nothing of their scale, which may be undefined)
                    add[r] = sum == 0.0f ? 0.0f : sum * inv * (low ? W_DOWN : 1.0f);
                }
                if (__any_sync(0xFFFFFFFFu, down[0] != 0.0f || down[1] != 0.0f)) {
                    const float corr[2] = {ex2(down[0]), ex2(down[1])};
                    l[nq][0] = smc_paged_fold(l[nq][0], down[0], 0.0f), l[nq][1] = smc_paged_fold(l[nq][1], down[1], 0.0f);
#pragma unroll
                    for (int i = 0; i < KS; ++i) o[nq][i][0] *= corr[0], o[nq][i][1] *= corr[1], o[nq][i][2] *= corr[0], o[nq][i][3] *= corr[1];
                }
                l[nq][0] += add[0], l[nq][1] += add[1];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float a = s[nq][j >> 1][2 * (j & 1)], b = s[nq][j >> 1][2 * (j & 1) + 1];
                    const uint32_t hi = half2_bits(a, b);
                    w[nq][0][j] = transposed(hi & seen);
                    if constexpr (SPLIT) w[nq][1][j] = transposed(rest_bits(a, b, hi) & seen);
                }
            }
            landed(half);
            // values that do not count are zeros whatever their bytes are: the weights there are 0, and codes may be undefined
            uint32_t keep[4] = {~0u, ~0u, ~0u, ~0u};
            if (now.tile0 < now.lo || now.tile0 + UNIT > now.hi) {
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (now.tile0 + 16 * t + e < now.lo || now.tile0 + 16 * t + e >= now.hi) keep[e >> 2] &= ~(0xFFu << (8 * (e & 3)));
            }
            const uint32_t vbase = ring + (uint32_t)((half % SLOTS) * R::SLOT + ((16 * t) >> c.shift) * ((HD << c.shift) + pad) + ((16 * t) & (page - 1)));
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                const uint4 ra = smc_lds128(vbase + (uint32_t)((16 * i + g) << c.shift)), rb = smc_lds128(vbase + (uint32_t)((16 * i + 8 + g) << c.shift));
                const uint32_t wa[4] = {ra.x & keep[0], ra.y & keep[1], ra.z & keep[2], ra.w & keep[3]}, wb[4] = {rb.x & keep[0], rb.y & keep[1], rb.z & keep[2], rb.w & keep[3]};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t a[4] = {smc_e4m3x2_half2(wa[k] & 0xFFFFu), smc_e4m3x2_half2(wb[k] & 0xFFFFu), smc_e4m3x2_half2(wa[k] >> 16), smc_e4m3x2_half2(wb[k] >> 16)};
#pragma unroll
                    for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
                        for (int pl = PL - 1; pl >= 0; --pl) mma_f16(o[nq][i], a, w[nq][pl][2 * k], w[nq][pl][2 * k + 1]);
                }
            }
            __syncwarp();
            request(later, false, half % SLOTS);
            ++half;
            now = next, next = later, sc_now = sc_next;
        }

        // ---- the segment's end: the warps' sums, eight rows at a time
        const bool whole = begin >= first && end <= last;
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq) {
            if (8 * nq >= pairs) continue;  // (the same for all)
            float sum[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                sum[r] = l[nq][r];
                sum[r] += __shfl_xor_sync(0xFFFFFFFFu, sum[r], 4);
                sum[r] += __shfl_xor_sync(0xFFFFFFFFu, sum[r], 8);
                sum[r] += __shfl_xor_sync(0xFFFFFFFFu, sum[r], 16);
            }
            // half of the dimensions at a time; warp w then adds rows 2 w, 2 w + 1 of all
#pragma unroll
            for (int part = 0; part < 2; ++part) {
                __syncthreads();
                float *row = merge + (warp * 8 + 2 * t) * R::MERGE_ROW;
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    if (part == 0 && g == 0) row[r * R::MERGE_ROW + HD / 2] = M[nq][r], row[r * R::MERGE_ROW + HD / 2 + 1] = sum[r];
#pragma unroll
                    for (int i = 0; i < KS / 2; ++i)
                        row[r * R::MERGE_ROW + 16 * i + g] = o[nq][part * (KS / 2) + i][r], row[r * R::MERGE_ROW + 16 * i + 8 + g] = o[nq][part * (KS / 2) + i][2 + r];
                }
                __syncthreads();
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float *rows = merge + (2 * warp + r) * R::MERGE_ROW;  // of warp v: + 8 v rows
                    const int m = 8 * nq + 2 * warp + r, pair = m0 + m, tok = pair / group;
                    if (m >= pairs) continue;
                    float top = -INFINITY, fac[WARPS], all = 0.0f;
#pragma unroll
                    for (int v = 0; v < WARPS; ++v) top = fmaxf(top, rows[v * 8 * R::MERGE_ROW + HD / 2]);
                    const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
                    for (int v = 0; v < WARPS; ++v) {
                        const float down = rows[v * 8 * R::MERGE_ROW + HD / 2] - ref;
                        fac[v] = ex2(down);
                        all = smc_paged_fold(rows[v * 8 * R::MERGE_ROW + HD / 2 + 1], down, all);
                    }
                    const float norm = whole ? (all == 0.0f ? 0.0f : 1.0f / all) : 1.0f;
                    float *part_row = partial(work, blockIdx.x, begin < first ? 0 : 1, PARTED ? PART : u.max_rows * group, HD) + (size_t)m * (HD + 4);
                    T *dst = static_cast<T *>(u.out) + ((size_t)(p.r0 + tok) * u.heads + h * group + pair - tok * group) * HD;
#pragma unroll
                    for (int i = 0; i < HD / 64; ++i) {
                        float a = 0.0f;
#pragma unroll
                        for (int v = 0; v < WARPS; ++v) a = fmaf(rows[v * 8 * R::MERGE_ROW + 32 * i + lane], fac[v], a);
                        const int d = part * (HD / 2) + 32 * i + lane;
                        if (whole) dst[d] = from_f<T>(a * norm);
                        else part_row[d] = a;
                    }
                    if (!whole && part == 0 && lane == 0) part_row[HD] = top, part_row[HD + 1] = all;
                }
            }
        }
        seg = stop;
    }
}

// One block of threads = one row and head: joins what the runs left of its segment.  Four dimensions a thread, the runs dealt to groups of threads, so that
// all loads go out at once; each group adds its runs in their order, then the groups' sums are added in theirs.  Latency bounds it: 16 rows 5.5 us from cold caches, 2048 7.4.
template <typename T, int HD, int JOIN_THREADS, bool PARTED>
__global__ void __launch_bounds__(JOIN_THREADS) paged_join_kernel(const smc_paged_view c, const smc_paged_query u, const float *__restrict__ work, int grid)
{
    constexpr int LANES = HD / 4, GROUPS = JOIN_THREADS / LANES;
    smc_grid_dep_sync();
    const int group = u.heads / c.kvh, most = u.max_rows * group, m = blockIdx.x % most, h = blockIdx.x / most % c.kvh, s = blockIdx.x / most / c.kvh, tid = threadIdx.x;
    __shared__ int part[2][JOIN_THREADS / 32];
    __shared__ float tops[JOIN_THREADS / 32], sums[JOIN_THREADS / 32], factor[RUNS_MOST];
    __shared__ float4 outs[GROUPS][LANES];
    int before = 0, units = 0;
    for (int i = tid; i < c.batch; i += JOIN_THREADS) {
        const int n = units_of<PARTED>(c, span_of<PARTED>(c, u, i));
        units += n;
        if (i < s) before += n;
    }
    before = __reduce_add_sync(0xFFFFFFFFu, before), units = __reduce_add_sync(0xFFFFFFFFu, units);
    if ((tid & 31) == 0) part[0][tid >> 5] = before, part[1][tid >> 5] = units;
    __syncthreads();
    before = 0, units = 0;
#pragma unroll
    for (int i = 0; i < JOIN_THREADS / 32; ++i) before += part[0][i], units += part[1][i];
    const Span p = span_of<PARTED>(c, u, s);
    if (m >= p.n * group) return;
    const int runs = min(grid, units), begin = before + (PARTED ? h * p.parts + m / PART : h) * p.tiles, c0 = run_of(begin, runs, units), count = run_of(begin + p.tiles - 1, runs, units) - c0 + 1;
    if (count == 1) return;  // whole in one run
    auto row = [&](int i) { return work + ((size_t)(c0 + i) * 2 + (i == 0)) * (PARTED ? PART : most) * (HD + 4) + (size_t)(PARTED ? m % PART : m) * (HD + 4); };
    float top = -INFINITY, sum_mine = 0.0f;
    for (int i = tid; i < count; i += JOIN_THREADS) {
        factor[i] = row(i)[HD];
        top = fmaxf(top, factor[i]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    if ((tid & 31) == 0) tops[tid >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < JOIN_THREADS / 32; ++i) top = fmaxf(top, tops[i]);
    const float ref = top == -INFINITY ? 0.0f : top;
    for (int i = tid; i < count; i += JOIN_THREADS) {
        const float down = factor[i] - ref;
        factor[i] = ex2(down);
        sum_mine = smc_paged_fold(row(i)[HD + 1], down, sum_mine);
    }
    const float sum_warp = smc_group_sum<32>(sum_mine);
    if ((tid & 31) == 0) sums[tid >> 5] = sum_warp;
    __syncthreads();
    const int g = tid / LANES, d = tid % LANES;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int i = g; i < count; i += GROUPS) {
        const float4 x = *reinterpret_cast<const float4 *>(row(i) + 4 * d);
        const float w = factor[i];
        o.x = fmaf(x.x, w, o.x), o.y = fmaf(x.y, w, o.y), o.z = fmaf(x.z, w, o.z), o.w = fmaf(x.w, w, o.w);
    }
    outs[g][d] = o;
    __syncthreads();
    if (tid < HD) {
        float sum = 0.0f, v = 0.0f;
#pragma unroll
        for (int i = 0; i < JOIN_THREADS / 32; ++i) sum += sums[i];
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) v += reinterpret_cast<const float *>(&outs[i][0])[tid];
        const int tok = m / group;
        static_cast<T *>(u.out)[((size_t)(p.r0 + tok) * u.heads + h * group + m - tok * group) * HD + tid] = from_f<T>(sum == 0.0f ? 0.0f : v / sum);
    }
}

template <int N> struct Dim {
    static constexpr int v = N;
};

// Whole segments to each CTA, and nothing left to join, or the units spread evenly over two CTAs an SM (four units, one a warp, to each where there are that few)?
// Whole: up to 8 tiles a segment (64 x 8 segments of 8: 18 us, spread 37), and up to 32 where there are four times as many segments (bf16, 4 rows a group, whole /
// spread: 16 tiles, 16 segments 13.1 / 12.3 us, 32 13.0 / 13.0, 64 13.1 / 17.5, 512 29 / 47; 32 tiles, 16 segments 20 / 13, 128 22 / 37, 512 45 / 55, 1024 81 / 81).
// Beyond, the longest segments are what the others wait for: 63 tiles, 1024 segments 148 / 123; 125 tiles, 512 segments 152 / 122.
constexpr int FEW_TILES = 8, SOME_TILES = 32;
int tiles_of(int max_len) { return max_len <= 0 ? 1 : (max_len - 1) / UNIT + 1; }
bool alone(long long segments, int max_len) { return tiles_of(max_len) <= FEW_TILES || (tiles_of(max_len) <= SOME_TILES && segments >= 4LL * tiles_of(max_len)); }
int parts_of(int pairs) { return (pairs + PART - 1) / PART; }
int runs_for(const smc_ctx *ctx, int kvh, int batch, int parts, int max_len)
{
    const long long segments = (long long)batch * kvh, most = std::min(2 * ctx->sm_count, RUNS_MOST);
    return (int)std::min(most, alone(segments, max_len) ? segments : (segments * parts * tiles_of(max_len) + WARPS - 1) / WARPS);
}

}  // namespace

// A part costs a pass over the keys, from L2 but for the first, where the tcgen05 form takes 256 pairs at once: up to four parts, and fifteen tiles of keys for each.
// Here / there in us, 8 KV heads of 128, sequences of up to so many keys:
//            one sequence         8                    24                   64
//   20 pairs  2000: 14 / 19, 8000: 22 / 26    2000: 28 / 44, 8000: 47 / 106    2000: 58 / 85, 8000: 129 / 264    2000: 109 / 158, 8000: 266 / 555
//   48        2000: 17 / 20, 8000: 27 / 27    2000: 34 / 44, 3000: 34 / 49     2000: 79 / 76, 3000:  87 / 123    2000: 161 / 165, 3000: 183 / 238
//   64        4000: 25 / 24, 8000: 30 / 28    2000: 37 / 42, 4000: 39 / 65     3000: 103 / 118, 4000: 140 / 153  3000: 262 / 224, 4000: 261 / 277
//   64 fp32   4000: 31 / 30, 8000: 37 / 34    2000: 45 / 45, 4000: 50 / 76     3000: 130 / 132, 4000: 178 / 170  3000: 333 / 251, 4000: 342 / 308, 6000: 377 / 429
// So 64 pairs of one sequence lose 1 to 3 us by the rule, and 64 fp32 ones of 64 sequences of some 4000 lose 34; few sequences with 33 and more pairs would gain from half as many tiles.
// Up to 16 pairs: 16, one sequence of 500 12 / 16 us, 64 of 8000 151 / 523.
bool smc_paged_decode_takes(int group, int max_rows, int max_len)
{
    const long long pairs = (long long)max_rows * group;
    return pairs <= PART || (pairs <= PART * PARTS_MOST && tiles_of(max_len) >= PART_TILES * (int)((pairs + PART - 1) / PART));
}

size_t smc_paged_decode_work(const smc_ctx *ctx, int kvh, int batch, int heads, int hd, int max_rows, int max_len)
{
    return alone((long long)batch * kvh, max_len) ? 0 : (size_t)runs_for(ctx, kvh, batch, parts_of(max_rows * (heads / kvh)), max_len) * 2 * std::min(PART, max_rows * (heads / kvh)) * (hd + 4) * sizeof(float);
}

int smc_launch_paged_decode(smc_ctx *ctx, const smc_paged_view &c, const smc_paged_query &u, float *work, cudaStream_t s)
{
    const int pairs = u.max_rows * (u.heads / c.kvh), runs = runs_for(ctx, c.kvh, c.batch, parts_of(pairs), u.max_len);
    const long long capacity = ((long long)c.width << c.shift) / UNIT + 2;  // (tiles that a sequence may have)
    if (capacity * parts_of(pairs) > 0x7FFFFFFF / ((long long)c.batch * c.kvh) || (long long)c.batch * c.kvh * pairs > 0x7FFFFFFF) return smc_fail(ctx, SMC_E_UNSUPPORTED, "paged_attention: %d sequences of %d heads in one call", c.batch, u.heads);
    // (few rows to join have many runs each: 512 threads a row, 23.3 us for the call of 32 rows over 30 001 keys, 128: 25.4; 2048 rows over 8000: 130 and 121)
    const bool whole = alone((long long)c.batch * c.kvh, u.max_len), many = (long long)c.batch * c.kvh * pairs >= 1024;
    auto pick = [&](auto type, auto hd, auto parted) {
        using T = decltype(type);
        constexpr int HD = decltype(hd)::v;
        constexpr bool PARTED = decltype(parted)::v != 0;
        auto main = paged_decode_kernel<T, HD, 2, PARTED>;
        if constexpr (!PARTED)
            if (pairs <= 8) main = paged_decode_kernel<T, HD, 1, false>;
        cudaFuncSetAttribute(main, cudaFuncAttributeMaxDynamicSharedMemorySize, Ring<HD>::SMEM);
        smc_launch_dep(ctx->use_pdl, main, dim3(runs), dim3(THREADS), Ring<HD>::SMEM, s, c, u, work, whole ? 1 : 0, ctx->d_status);
        if (whole || runs == 1) return;
        const dim3 grid((unsigned)(c.batch * c.kvh * pairs));
        if (many) smc_launch_dep(ctx->use_pdl, paged_join_kernel<T, HD, 128, PARTED>, grid, dim3(128), 0, s, c, u, work, runs);
        else smc_launch_dep(ctx->use_pdl, paged_join_kernel<T, HD, 512, PARTED>, grid, dim3(512), 0, s, c, u, work, runs);
    };
    auto form = [&](auto type, auto hd) { pairs > PART ? pick(type, hd, Dim<1>()) : pick(type, hd, Dim<0>()); };
    if (u.bf16) u.hd == 128 ? form(bf16(), Dim<128>()) : form(bf16(), Dim<64>());
    else u.hd == 128 ? form(float(), Dim<128>()) : form(float(), Dim<64>());
    SMC_LAUNCH_CHECK(ctx);
    return SMC_OK;
}
