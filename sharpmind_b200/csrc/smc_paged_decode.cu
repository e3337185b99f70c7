// Attention of a few rows of every sequence over the paged cache (a decode step, drafts): the whole cache passes once through registers, so HBM is
// the bound, and the work has to be even over the device whatever the sequences' lengths are.
//
// Units of 64 keys of one sequence and KV head, in the order (sequence, head, tile); the grid's CTAs take equal runs of them, a CTA's four
// warps take its units in turn.  What a CTA has of one sequence and head (a segment) is merged in shared memory at its end; a segment that a run's
// border cuts leaves as (running maximum, sum, unnormalised output), and a second small kernel joins those.  The order of all sums is fixed by the lengths.
//
// A warp's unit: keys and values arrive by bulk copies in a ring of its own, K and V of 64 tokens a slot, two slots ahead.  Scores and outputs
// are mma.sync m16n8k16 in fp16 with fp32 sums: an e4m3 code is exact in fp16, the queries are scaled by a power of two per row to 2^15 at most.  bfloat16
// queries are exact so, 16 (row, head) pairs a tile; fp32 ones go in as hi + lo, 22 bits, in the tile's upper and lower eight rows, which costs
// nothing where eight pairs are all there are.  Both products' contraction indices are permuted so that a thread reads 16 contiguous codes:
// thread t of a quad owns dims [16 t, 16 t + 16) (and + 64) of the keys, and tokens [16 t, 16 t + 16) of scores, weights and values, which
// lie in one page, so a unit's scales are two numbers a thread.
//   y_j = x_j log2(e) + log2(s_v);  w_j = 2^(y_j - M), M the running maximum of y less 14;  O = sum w_j code_j;  l = sum w_j / s_v;  out = O / l
// The value scales ride in the exponent, so the weights stay within fp16 whatever the scales are: 2^14 at most, and 2^-38 of that still counts.
#include "smc_async.cuh"
#include "smc_paged.cuh"

namespace {

constexpr int WARPS = 4, THREADS = 32 * WARPS, UNIT = 64, SLOTS = 3, CHUNKS = 256;
constexpr float W_SHIFT = 14.0f;

template <int HD>
struct Ring {
    static constexpr int SLOT = UNIT * HD + 128;               // values of 16- and 32-token pages lie 32 and 64 bytes further apart: no bank conflicts
    static constexpr int OFF_MERGE = WARPS * SLOTS * SLOT;      // [warps 1 ..][8 rows][HD + 4] floats
    static constexpr int MERGE_ROW = HD + 4;                    // O, then maximum and sum
    static constexpr int OFF_BAR = OFF_MERGE + (WARPS - 1) * 8 * MERGE_ROW * 4, OFF_PLAN = OFF_BAR + WARPS * SLOTS * 8;
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

// tiles [t0, t0 + tiles) of 64 keys that rows of sequence s see; one tile, all masked, where there is no key, none where there is no row
struct Span {
    int r0, n, len, from, t0, tiles;
    bool bad;
};
__device__ __forceinline__ Span span_of(const smc_paged_view &c, const smc_paged_query &u, int s)
{
    const smc_paged_seq sq = smc_paged_sequence(c, s);
    Span p;
    p.r0 = sq.r0, p.n = min(sq.n, u.max_rows), p.len = sq.len, p.bad = sq.bad || sq.n > u.max_rows;
    p.from = u.window > 0 ? max(0, sq.len - p.n + 1 - u.window) : 0;
    p.t0 = p.from / UNIT;
    p.tiles = p.n == 0 ? 0 : max(1, (sq.len + UNIT - 1) / UNIT - p.t0);
    return p;
}
// run of units of CTA i of n: [first, first of the next)
__device__ __forceinline__ int run_first(int i, int n, int units) { return (int)((long long)i * units / n); }
__device__ __forceinline__ int run_of(int unit, int n, int units) { return (int)(((long long)(unit + 1) * n - 1) / units); }

// Where a warp is among the units: sequence s has [base, base + kvh * tiles)
struct Place {
    int s, base;
    Span p;
};
__device__ __forceinline__ void advance(const smc_paged_view &c, const smc_paged_query &u, Place &w, int unit)
{
    while (w.base + c.kvh * w.p.tiles <= unit && w.s + 1 < c.batch) {
        w.base += c.kvh * w.p.tiles;
        w.p = span_of(c, u, ++w.s);
    }
}

// slot of a CTA's cut segment: 0 where it began before the run, 1 where it begins in it
__device__ __forceinline__ float *partial(float *work, int cta, int which, int rows, int hd) { return work + ((size_t)cta * 2 + which) * rows * (hd + 4); }

template <typename T, int HD, int MT>
__global__ void __launch_bounds__(THREADS, 2) paged_decode_kernel(const smc_paged_view c, const smc_paged_query u, float *work, int *status)
{
    constexpr bool SPLIT = sizeof(T) == 4;          // queries and weights as hi + lo
    constexpr int ROWS = SPLIT ? 8 : 16, KS = HD / 16, CH = HD / 64, NT = HD / 8, OCT = SPLIT ? 1 : 2;
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
            const Span p = span_of(c, u, s);
            n += c.kvh * p.tiles;
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
    const int runs = min((int)gridDim.x, units);  // (no run between two others is empty)
    if ((int)blockIdx.x >= runs) return;
    const int first = run_first(blockIdx.x, runs, units), last = run_first(blockIdx.x + 1, runs, units);
    Place at;
    {
        int lo = 0, hi = CHUNKS;  // the last group that starts at or before `first`
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (plan[mid] <= first) lo = mid;
            else hi = mid;
        }
        // (groups behind the last sequence start at `units`)
        at.s = min(lo * per, c.batch - 1), at.base = plan[lo], at.p = span_of(c, u, at.s);
        advance(c, u, at, first);
    }

    // ---- what is on its way: half-stages K, V of this warp's units first + warp, + 4, ...
    const int page = 1 << c.shift, pad = c.shift == 4 ? 32 : c.shift == 5 ? 64 : 0;
    struct Fetch {
        int tile0, h, id, lo, hi;  // the unit's first key, its head, the page of this thread's 16 tokens (-1: nothing to bring); keys that count
    };
    Place ahead = at;
    auto look = [&](int unit) {
        Fetch f{0, 0, -1, 0, 0};
        if (unit >= last) return f;
        advance(c, u, ahead, unit);
        const int rest = unit - ahead.base, h = rest / ahead.p.tiles;
        f.h = h, f.tile0 = (ahead.p.t0 + rest - h * ahead.p.tiles) * UNIT;
        f.lo = ahead.p.from, f.hi = ahead.p.len;
        const int key = f.tile0 + 16 * t, p0 = key >> c.shift << c.shift;
        if (p0 + page > f.lo && p0 < f.hi) {  // (pages that left the window may have gone to another sequence)
            f.id = smc_paged_page(c, ahead.s, key >> c.shift);
            if (f.id < 0) *status = SMC_STATUS_PAGED;
        }
        return f;
    };
    auto scales_of = [&](const Fetch &f) {
        return f.id < 0 ? make_float2(0.0f, 1.0f) : *reinterpret_cast<const float2 *>(c.scales + 2 * ((size_t)f.id * c.kvh + f.h));
    };
    const bool leader = g == 0 && ((16 * t) & (page - 1)) == 0;
    auto request = [&](const Fetch &f, bool values, int slot) {
        const bool bring = leader && f.id >= 0;
        const unsigned who = __ballot_sync(0xFFFFFFFFu, bring);
        if (lane == 0) smc_mbar_expect_tx(bars + 8 * slot, (uint32_t)(__popc(who) * page * HD));
        __syncwarp();
        if (bring) {
            const size_t block = ((size_t)f.id * c.kvh + f.h) * ((size_t)HD << c.shift);
            const uint32_t dst = ring + (uint32_t)(slot * R::SLOT + 16 * t * HD + (values ? ((16 * t) >> c.shift) * pad : 0));
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
        advance(c, u, at, seg);
        const Span p = at.p;
        const int h = (seg - at.base) / p.tiles, begin = at.base + h * p.tiles, end = begin + p.tiles, stop = min(end, last);
        const int pairs = p.n * group;
        uint32_t q[MT][KS][4];
        float rowf[MT][OCT];
        int pos[MT][OCT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int o = 0; o < OCT; ++o) {
                const int m = min(mt * ROWS + 8 * o + g, pairs - 1), i = m / group;  // (rows behind the last repeat it and are not stored)
                pos[mt][o] = p.len - p.n + i;
                const T *src = static_cast<const T *>(u.q) + (long long)(p.r0 + i) * u.q_stride + (size_t)(h * group + m - i * group) * HD + 16 * t;
                float x[4 * KS];
                float most = 0.0f;
#pragma unroll
                for (int e = 0; e < KS; ++e) {  // dims 64 (e / 4) + 16 t + 4 (e % 4)
                    float v[4];
                    smc_paged_load4(src + 64 * (e >> 2) + 4 * (e & 3), v);
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[4 * e + j] = v[j], most = fmaxf(most, fabsf(v[j]));
                }
                most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 2));
                // the largest magnitude goes to [2^14, 2^15)
                const int up = min(14 - ((int)(__float_as_uint(most) >> 23) - 127), 126);
                const float fac = __uint_as_float((uint32_t)(up + 127) << 23);
                rowf[mt][o] = u.scale * 1.44269504088896341f * __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
                for (int e = 0; e < KS; ++e) {
                    const uint32_t a = half2_bits(x[4 * e] * fac, x[4 * e + 1] * fac), b = half2_bits(x[4 * e + 2] * fac, x[4 * e + 3] * fac);
                    if constexpr (SPLIT) {
                        q[mt][e][0] = a, q[mt][e][2] = b;
                        q[mt][e][1] = rest_bits(x[4 * e] * fac, x[4 * e + 1] * fac, a), q[mt][e][3] = rest_bits(x[4 * e + 2] * fac, x[4 * e + 3] * fac, b);
                    } else {
                        q[mt][e][o] = a, q[mt][e][2 + o] = b;
                    }
                }
            }
        float o[MT][NT][4] = {}, M[MT][OCT], l[MT][OCT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < OCT; ++i) M[mt][i] = -INFINITY, l[mt][i] = 0.0f;

        for (; unit < stop; unit += WARPS) {
            const int key0 = now.tile0 + 16 * t;  // this thread's tokens of scores and values
            later = look(unit + 2 * WARPS);
            sc_next = scales_of(next);
            const bool here = now.id >= 0;
            // (a power of two's exponent; a scale that is none, left where no page is or undefined, stays what it is)
            const float bias = sc_now.y == sc_now.y ? (float)((int)(__float_as_uint(sc_now.y) >> 23) - 127) : sc_now.y, inv = 1.0f / sc_now.y;
            const bool inner = now.tile0 >= now.lo && now.tile0 + UNIT <= p.len - p.n + 1 && (u.window <= 0 || now.tile0 > p.len - 1 - u.window);
            uint32_t w[MT][4][4];  // weights as A fragments
            landed(half);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                float s[8][4] = {};
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t row = ring + (uint32_t)((half % SLOTS) * R::SLOT + (16 * (g >> 1) + 2 * j + (g & 1)) * HD + 16 * t);
#pragma unroll
                    for (int ch = 0; ch < CH; ++ch) {
                        const uint4 raw = smc_lds128(row + 64 * ch);
                        const uint32_t k4[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) mma_f16(s[j], q[mt][4 * ch + e], smc_e4m3x2_half2(k4[e] & 0xFFFFu), smc_e4m3x2_half2(k4[e] >> 16));
                    }
                }
                float y[OCT][16];
#pragma unroll
                for (int i = 0; i < OCT; ++i) {
                    const float f = rowf[mt][i] * sc_now.x;
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const float acc = SPLIT ? s[j >> 1][j & 1] + s[j >> 1][2 + (j & 1)] : s[j >> 1][2 * i + (j & 1)];
                        y[i][j] = fmaf(acc, f, bias);
                    }
                    if (!inner) {
                        const int hi = min(pos[mt][i], p.len - 1), lo = u.window > 0 ? pos[mt][i] - u.window : -1;
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            if (key0 + j > hi || key0 + j <= lo) y[i][j] = -INFINITY;
                    }
                    float top = y[i][0];
#pragma unroll
                    for (int j = 1; j < 16; ++j) top = fmaxf(top, y[i][j]);
                    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                    const float nm = fmaxf(M[mt][i], top - W_SHIFT), ref = nm == -INFINITY ? 0.0f : nm;
                    const float corr = ex2(M[mt][i] - ref);  // (-inf: nothing yet, 0)
                    M[mt][i] = nm;
                    float sum = 0.0f;
#pragma unroll
                    for (int j = 0; j < 16; ++j) sum += y[i][j] = ex2(y[i][j] - ref);
                    // (a row that sees none of these tokens takes nothing of their scale, which may be undefined)
                    l[mt][i] = fmaf(l[mt][i], corr, sum == 0.0f ? 0.0f : sum * inv);
                    if (__any_sync(0xFFFFFFFFu, corr != 1.0f)) {
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            o[mt][n][2 * i] *= corr, o[mt][n][2 * i + 1] *= corr;
                            if (SPLIT) o[mt][n][2] *= corr, o[mt][n][3] *= corr;
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int j = 4 * k + 2 * e;
                        if constexpr (SPLIT) {
                            w[mt][k][2 * e] = half2_bits(y[0][j], y[0][j + 1]);
                            w[mt][k][2 * e + 1] = rest_bits(y[0][j], y[0][j + 1], w[mt][k][2 * e]);
                        } else {
                            w[mt][k][2 * e] = half2_bits(y[0][j], y[0][j + 1]);
                            w[mt][k][2 * e + 1] = half2_bits(y[OCT - 1][j], y[OCT - 1][j + 1]);
                        }
                    }
            }
            __syncwarp();
            request(next, true, half % SLOTS);
            ++half;
            landed(half);
            // values that do not count are zeros whatever their bytes are: the weights there are 0, and codes may be undefined
            uint32_t keep[4] = {~0u, ~0u, ~0u, ~0u};
            if (now.tile0 < now.lo || now.tile0 + UNIT > now.hi || !__all_sync(0xFFFFFFFFu, here)) {
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (key0 + e < now.lo || key0 + e >= now.hi || !here) keep[e >> 2] &= ~(0xFFu << (8 * (e & 3)));
            }
            const uint32_t vbase = ring + (uint32_t)((half % SLOTS) * R::SLOT + ((16 * t) >> c.shift) * ((HD << c.shift) + pad) + ((16 * t) & (page - 1)));
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const uint4 raw = smc_lds128(vbase + (uint32_t)((8 * n + g) << c.shift));
                const uint32_t v4[4] = {raw.x & keep[0], raw.y & keep[1], raw.z & keep[2], raw.w & keep[3]};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t b0 = smc_e4m3x2_half2(v4[k] & 0xFFFFu), b1 = smc_e4m3x2_half2(v4[k] >> 16);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) mma_f16(o[mt][n], w[mt][k], b0, b1);
                }
            }
            __syncwarp();
            request(later, false, half % SLOTS);
            ++half;
            now = next, next = later, sc_now = sc_next;
        }

        // ---- the segment's end: warps 1 .. leave what they have, warp 0 joins it, eight rows at a time
        const bool whole = begin >= first && end <= last;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < OCT; ++i) {
                if (mt * ROWS + 8 * i >= pairs) continue;  // (the same for all)
                float sum = l[mt][i];
                sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 1);
                sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 2);
                __syncthreads();
                if (warp > 0) {
                    float *row = merge + ((warp - 1) * 8 + g) * R::MERGE_ROW;
                    if (t == 0) row[HD] = M[mt][i], row[HD + 1] = sum;
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                        *reinterpret_cast<float2 *>(row + 8 * n + 2 * t) =
                            SPLIT ? make_float2(o[mt][n][0] + o[mt][n][2], o[mt][n][1] + o[mt][n][3]) : make_float2(o[mt][n][2 * i], o[mt][n][2 * i + 1]);
                }
                __syncthreads();
                if (warp == 0) {
                    float top = M[mt][i];
#pragma unroll
                    for (int v = 0; v < WARPS - 1; ++v) top = fmaxf(top, merge[(v * 8 + g) * R::MERGE_ROW + HD]);
                    const float ref = top == -INFINITY ? 0.0f : top;
                    float fac[WARPS];
                    fac[0] = ex2(M[mt][i] - ref);
                    sum *= fac[0];
#pragma unroll
                    for (int v = 0; v < WARPS - 1; ++v) {
                        const float *row = merge + (v * 8 + g) * R::MERGE_ROW;
                        fac[v + 1] = ex2(row[HD] - ref);
                        sum = fmaf(row[HD + 1], fac[v + 1], sum);
                    }
                    const int m = mt * ROWS + 8 * i + g, tok = m / group;
                    const float norm = whole ? (sum == 0.0f ? 0.0f : 1.0f / sum) : 1.0f;
                    float *part = partial(work, blockIdx.x, begin < first ? 0 : 1, u.max_rows * group, HD) + (size_t)m * (HD + 4);
                    T *dst = static_cast<T *>(u.out) + ((size_t)(p.r0 + tok) * u.heads + h * group + m - tok * group) * HD;
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float a = (SPLIT ? o[mt][n][0] + o[mt][n][2] : o[mt][n][2 * i]) * fac[0], b = (SPLIT ? o[mt][n][1] + o[mt][n][3] : o[mt][n][2 * i + 1]) * fac[0];
#pragma unroll
                        for (int v = 0; v < WARPS - 1; ++v) {
                            const float2 x = *reinterpret_cast<const float2 *>(merge + (v * 8 + g) * R::MERGE_ROW + 8 * n + 2 * t);
                            a = fmaf(x.x, fac[v + 1], a), b = fmaf(x.y, fac[v + 1], b);
                        }
                        a *= norm, b *= norm;
                        if (m < pairs) {
                            if (!whole) *reinterpret_cast<float2 *>(part + 8 * n + 2 * t) = make_float2(a, b);
                            else if constexpr (SPLIT) *reinterpret_cast<float2 *>(dst + 8 * n + 2 * t) = make_float2(a, b);
                            else *reinterpret_cast<uint32_t *>(dst + 8 * n + 2 * t) = pack2(a, b);
                        }
                    }
                    if (!whole && m < pairs && t == 0) part[HD] = top, part[HD + 1] = sum;
                }
            }
        seg = stop;
    }
}

// One block of threads = one row and head: joins what the runs left of its segment.  Four dimensions a thread, the runs dealt to groups of threads, so that
// all loads go out at once; each group adds its runs in their order, then the groups' sums are added in theirs.
constexpr int JOIN_THREADS = 512;
template <typename T, int HD>
__global__ void __launch_bounds__(JOIN_THREADS) paged_join_kernel(const smc_paged_view c, const smc_paged_query u, const float *__restrict__ work, int grid)
{
    constexpr int LANES = HD / 4, GROUPS = JOIN_THREADS / LANES;
    smc_grid_dep_sync();
    const int group = u.heads / c.kvh, most = u.max_rows * group, m = blockIdx.x % most, h = blockIdx.x / most % c.kvh, s = blockIdx.x / most / c.kvh, tid = threadIdx.x;
    __shared__ int part[2][JOIN_THREADS / 32];
    __shared__ float tops[JOIN_THREADS / 32], sums[JOIN_THREADS / 32], factor[JOIN_THREADS];
    __shared__ float4 outs[GROUPS][LANES];
    int before = 0, units = 0;
    for (int i = tid; i < c.batch; i += JOIN_THREADS) {
        const int n = c.kvh * span_of(c, u, i).tiles;
        units += n;
        if (i < s) before += n;
    }
    before = __reduce_add_sync(0xFFFFFFFFu, before), units = __reduce_add_sync(0xFFFFFFFFu, units);
    if ((tid & 31) == 0) part[0][tid >> 5] = before, part[1][tid >> 5] = units;
    __syncthreads();
    before = 0, units = 0;
#pragma unroll
    for (int i = 0; i < JOIN_THREADS / 32; ++i) before += part[0][i], units += part[1][i];
    const Span p = span_of(c, u, s);
    if (m >= p.n * group) return;
    const int runs = min(grid, units), begin = before + h * p.tiles, c0 = run_of(begin, runs, units), count = run_of(begin + p.tiles - 1, runs, units) - c0 + 1;
    if (count == 1) return;  // whole in one run
    auto row = [&](int i) { return work + ((size_t)(c0 + i) * 2 + (i == 0)) * most * (HD + 4) + (size_t)m * (HD + 4); };
    // (one thread a run: a grid has no more than two an SM)
    const float mine = tid < count ? row(tid)[HD] : -INFINITY, sum_mine = tid < count ? row(tid)[HD + 1] : 0.0f;
    float top = mine;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    if ((tid & 31) == 0) tops[tid >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < JOIN_THREADS / 32; ++i) top = fmaxf(top, tops[i]);
    const float f = ex2(mine - (top == -INFINITY ? 0.0f : top));
    factor[tid] = f;
    const float sum_warp = smc_group_sum<32>(tid < count ? sum_mine * f : 0.0f);
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

// CTAs: two an SM, but four units (one a warp) each where there are that few
int runs_for(const smc_ctx *ctx, int kvh, int batch, int max_len)
{
    const long long bound = (long long)batch * kvh * std::max(1, (max_len + UNIT - 1) / UNIT);
    return (int)std::min<long long>(std::min(2 * ctx->sm_count, JOIN_THREADS), (bound + WARPS - 1) / WARPS);
}

}  // namespace

bool smc_paged_decode_takes(int bf16, int group, int max_rows) { return (long long)max_rows * group <= (bf16 ? 32 : 16); }

size_t smc_paged_decode_work(const smc_ctx *ctx, int kvh, int batch, int heads, int hd, int max_rows, int max_len)
{
    return (size_t)runs_for(ctx, kvh, batch, max_len) * 2 * max_rows * (heads / kvh) * (hd + 4) * sizeof(float);
}

int smc_launch_paged_decode(smc_ctx *ctx, const smc_paged_view &c, const smc_paged_query &u, float *work, cudaStream_t s)
{
    const int pairs = u.max_rows * (u.heads / c.kvh), runs = runs_for(ctx, c.kvh, c.batch, u.max_len);
    auto go = [&](auto main, auto join, int smem) {
        cudaFuncSetAttribute(main, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        smc_launch_dep(ctx->use_pdl, main, dim3(runs), dim3(THREADS), smem, s, c, u, work, ctx->d_status);
        if (runs > 1) smc_launch_dep(ctx->use_pdl, join, dim3((unsigned)(c.batch * c.kvh * pairs)), dim3(JOIN_THREADS), 0, s, c, u, work, runs);
    };
    if (u.bf16) {
        if (u.hd == 128) pairs <= 16 ? go(paged_decode_kernel<bf16, 128, 1>, paged_join_kernel<bf16, 128>, Ring<128>::SMEM) : go(paged_decode_kernel<bf16, 128, 2>, paged_join_kernel<bf16, 128>, Ring<128>::SMEM);
        else pairs <= 16 ? go(paged_decode_kernel<bf16, 64, 1>, paged_join_kernel<bf16, 64>, Ring<64>::SMEM) : go(paged_decode_kernel<bf16, 64, 2>, paged_join_kernel<bf16, 64>, Ring<64>::SMEM);
    } else {
        if (u.hd == 128) pairs <= 8 ? go(paged_decode_kernel<float, 128, 1>, paged_join_kernel<float, 128>, Ring<128>::SMEM) : go(paged_decode_kernel<float, 128, 2>, paged_join_kernel<float, 128>, Ring<128>::SMEM);
        else pairs <= 8 ? go(paged_decode_kernel<float, 64, 1>, paged_join_kernel<float, 64>, Ring<64>::SMEM) : go(paged_decode_kernel<float, 64, 2>, paged_join_kernel<float, 64>, Ring<64>::SMEM);
    }
    SMC_LAUNCH_CHECK(ctx);
    return SMC_OK;
}
