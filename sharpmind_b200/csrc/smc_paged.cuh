// What the kernels of the paged key/value cache share: the cache and its sequences as kernels see them, rows and positions, and the 8-bit codes.
#pragma once
#include <cuda_fp8.h>

#include "smc_mma.cuh"

// status word of smc_device_status: a page number, length or position outside of what the call was given
constexpr int SMC_STATUS_PAGED = 6;

struct smc_paged_view {
    uint8_t *k, *v;  // [pages, kvh, page, hd], [pages, kvh, hd, page] e4m3 codes
    float *scales;   // [pages, kvh, 2]
    int pages, kvh, shift;  // page = 1 << shift
    const int *table, *lengths, *row_start;
    int batch, width, rows;
};

#ifdef __CUDACC__
// Rows [r0, r0 + n) of sequence s sit at positions [len - n, len); whatever the device arrays hold, rows stay inside of [0, rows) and
// positions inside of the table.
struct smc_paged_seq {
    int r0, n, len;
    bool bad;
};
__device__ __forceinline__ smc_paged_seq smc_paged_sequence(const smc_paged_view &c, int s)
{
    smc_paged_seq q;
    int a = s, b = s + 1;
    if (c.row_start) a = c.row_start[s], b = c.row_start[s + 1];
    q.r0 = min(max(a, 0), c.rows);
    q.n = min(max(b, q.r0), c.rows) - q.r0;
    const int len = c.lengths[s];
    const long long most = min((long long)c.width << c.shift, 0x7FFFFF00LL);  // (a few tiles of keys behind a length are still an int)
    q.len = (int)min((long long)max(len, 0), most);
    q.bad = a < 0 || b < a || b > c.rows || len < 0 || len > most;
    return q;
}
// page `i` of sequence s, or -1
__device__ __forceinline__ int smc_paged_page(const smc_paged_view &c, int s, int i)
{
    const int id = i < c.width ? c.table[(size_t)s * c.width + i] : -1;
    return id >= 0 && id < c.pages ? id : -1;
}
// the sequence that row r of the call belongs to (-1: a row behind the last one)
__device__ __forceinline__ int smc_paged_row_sequence(const smc_paged_view &c, int r)
{
    if (!c.row_start) return r < c.batch ? r : -1;
    int lo = 0, hi = c.batch;  // the last s with row_start[s] <= r
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (c.row_start[mid] <= r) lo = mid;
        else hi = mid;
    }
    return c.row_start[lo] <= r && r < c.row_start[lo + 1] ? lo : -1;
}

// two codes as halves (exact: e4m3 is a subset of fp16)
__device__ __forceinline__ uint32_t smc_e4m3x2_half2(uint32_t two)
{
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((unsigned short)two));
    return h;
}
__device__ __forceinline__ void smc_e4m3x4_float(uint32_t w, float (&f)[4])
{
    const uint32_t a = smc_e4m3x2_half2(w & 0xFFFFu), b = smc_e4m3x2_half2(w >> 16);
    const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&a)), y = __half22float2(*reinterpret_cast<const __half2 *>(&b));
    f[0] = x.x, f[1] = x.y, f[2] = y.x, f[3] = y.y;
}
// four values as codes, round to nearest even; the first in the low byte
__device__ __forceinline__ uint32_t smc_float_e4m3x4(const float (&f)[4])
{
    unsigned short a, b;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(a) : "f"(f[1]), "f"(f[0]));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(b) : "f"(f[3]), "f"(f[2]));
    return (uint32_t)a | ((uint32_t)b << 16);
}
// A weight carries its value's scale, w = 2^(y - R), y = x + log2 s_v, and the softmax's sum is l = sum 2^(x - R) = sum w / s_v.  Scales are 2^-40 .. 2^120 and the
// largest y is at most 16 above R, so of the keys of a row the one with the largest x has 2^(x - R) >= 2^-120, while its w, and the factor that brings an earlier sum
// to a new R, may be smaller than fp32 holds (2^-126): both attention forms keep the sum from losing it.
__device__ __forceinline__ int smc_paged_log2(float scale) { return (int)(__float_as_uint(scale) >> 23) - 127; }  // of a power of two; 128 of an undefined one
// l 2^d + add for d <= 0; 2^d itself may vanish where l 2^d counts
__device__ __forceinline__ float smc_paged_fold(float l, float d, float add)
{
    float f = ex2(d);
    if (d < -100.0f) f = ex2(0.5f * d), l *= f;
    return fmaf(l, f, add);
}
// Four neighbouring elements of a row as floats, and floats as elements
template <typename T> __device__ __forceinline__ void smc_paged_load4(const T *p, float (&f)[4]) { load_v<T, 4>(p, f); }
template <typename T> __device__ __forceinline__ void smc_paged_store4(T *p, const float (&f)[4]) { store_v<T, 4>(p, f); }
#endif

// Launchers of the attention's forms: a few rows of every sequence (smc_paged_decode.cu), or many (smc_paged_prompt.cu)
struct smc_paged_query {
    const void *q;
    long long q_stride;
    void *out;
    int bf16, heads, hd, window, max_rows, max_len;
    float scale;
};
bool smc_paged_decode_takes(int group, int max_rows, int max_len);
size_t smc_paged_decode_work(const smc_ctx *, int kvh, int batch, int heads, int hd, int max_rows, int max_len);
int smc_launch_paged_decode(smc_ctx *, const smc_paged_view &, const smc_paged_query &, float *work, cudaStream_t s);
size_t smc_paged_prompt_work(const smc_ctx *, int kvh, int batch, int rows, int heads, int hd, int max_len);
int smc_launch_paged_prompt(smc_ctx *, const smc_paged_view &, const smc_paged_query &, float *work, cudaStream_t s);
