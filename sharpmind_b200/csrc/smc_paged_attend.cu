// Causal attention over the paged cache: x_ij = scale q_i . k_j for the keys j <= p_i (window > 0: j > p_i - window) of a row's sequence, out_i =
// sum_j softmax(x_i)_j v_j, zeros for a row that sees no key.  One warp a row and head, one pass over the keys with the running maximum and sum.
#include "smc_paged.cuh"

namespace {

template <typename T, int HD>
__global__ void __launch_bounds__(128) paged_attend_kernel(const smc_paged_view c, const smc_paged_query u, int *status)
{
    smc_grid_dep_sync();
    constexpr int E = HD / 32;
    const int lane = threadIdx.x & 31;
    const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (w >= (long long)c.rows * u.heads) return;
    const int r = (int)(w / u.heads), hq = (int)(w % u.heads), h = hq / (u.heads / c.kvh);
    const int s = smc_paged_row_sequence(c, r);
    if (s < 0) return;
    const smc_paged_seq sq = smc_paged_sequence(c, s);
    if ((sq.bad || sq.n > u.max_rows) && lane == 0) *status = SMC_STATUS_PAGED;
    const int pos = sq.len - sq.n + r - sq.r0, end = pos + 1, from = u.window > 0 ? max(0, end - u.window) : 0;
    float q[E], o[E] = {}, m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) q[e] = to_f(static_cast<const T *>(u.q)[(long long)r * u.q_stride + (size_t)hq * HD + lane * E + e]) * u.scale;
    for (int j = from; j < end; ++j) {
        const int id = smc_paged_page(c, s, j >> c.shift), t = j & ((1 << c.shift) - 1);
        if (id < 0) {
            if (lane == 0) *status = SMC_STATUS_PAGED;
            continue;
        }
        const size_t block = (size_t)id * c.kvh + h;
        const uint8_t *k = c.k + ((block << c.shift) + t) * HD + lane * E, *v = c.v + ((block * HD + lane * E) << c.shift) + t;
        float x = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            float f[4];
            smc_e4m3x4_float(k[e], f);
            x = fmaf(q[e], f[0], x);
        }
        x = smc_group_sum<32>(x) * c.scales[2 * block];
        const float nm = fmaxf(m, x), corr = expf(m - nm), p = expf(x - nm), pv = p * c.scales[2 * block + 1];
        l = fmaf(l, corr, p), m = nm;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            float f[4];
            smc_e4m3x4_float(v[(size_t)e << c.shift], f);
            o[e] = fmaf(o[e], corr, pv * f[0]);
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) static_cast<T *>(u.out)[((size_t)r * u.heads + hq) * HD + lane * E + e] = from_f<T>(end > from ? o[e] / l : 0.0f);
}

}  // namespace

int smc_launch_paged_attend(smc_ctx *ctx, const smc_paged_view &c, const smc_paged_query &u, cudaStream_t s)
{
    const long long grid = ((long long)c.rows * u.heads + 3) / 4;
    if (grid > 0x7FFFFFFF) return smc_fail(ctx, SMC_E_UNSUPPORTED, "paged_attention: %d rows in one call", c.rows);
    auto go = [&](auto kernel) { smc_launch_dep(ctx->use_pdl, kernel, dim3((unsigned)grid), dim3(128), 0, s, c, u, ctx->d_status); };
    if (u.bf16) u.hd == 128 ? go(paged_attend_kernel<bf16, 128>) : go(paged_attend_kernel<bf16, 64>);
    else u.hd == 128 ? go(paged_attend_kernel<float, 128>) : go(paged_attend_kernel<float, 64>);
    SMC_LAUNCH_CHECK(ctx);
    return SMC_OK;
}
