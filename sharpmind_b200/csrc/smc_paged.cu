// The paged key/value cache: entry points, the update that rotates, quantises and places new tokens, and the read that turns pages back into
// values.  The attention over it: smc_paged_decode.cu, smc_paged_prompt.cu.
//
// A block is the tokens of one page and head, keys and values apart.  Its scale is 2^k, k = min{k >= -40 : amax <= 448 2^k}, amax over all that
// entered the block since its first token; a value is held as code = e4m3(x / scale) and stands for code * scale.  Dividing by a power of two is exact, so
// a code is off by half a step of e4m3, 2^-4 of the value, and a block whose scale grows loses only what falls under the smallest code: rounding an
// e4m3 number again after a change of its exponent changes nothing else.
// A block that a value without a finite magnitude entered has the scale NaN: rows that see one of its tokens come out as NaN, others do not.
#include "smc_paged.cuh"

namespace {

constexpr int UPDATE_THREADS = 128;
constexpr int SCALE_FLOOR = -40;

struct Update {
    smc_paged_view c;
    const void *k, *v, *q;
    void *q_out;
    long long k_stride, v_stride, q_stride;
    int heads, rope_dim, table_rows, neox, items;
    const float *cosT, *sinT;
    int *status;
};

// four rotated neighbours of head `x` at dimension d; c, s: the position's rows of the tables
template <typename T>
__device__ __forceinline__ void rotated4(const T *x, int d, int rope_dim, bool neox, const float *c, const float *s, float (&y)[4])
{
    smc_paged_load4(x + d, y);
    if (!c || d >= rope_dim) return;
    const int half = rope_dim >> 1;
    if (neox) {  // (i, i + half): half is a multiple of four
        float p[4];
        const bool low = d < half;
        const int i = low ? d : d - half;
        smc_paged_load4(x + (low ? d + half : d - half), p);
        const float4 cc = *reinterpret_cast<const float4 *>(c + i), ss = *reinterpret_cast<const float4 *>(s + i);
        const float ca[4] = {cc.x, cc.y, cc.z, cc.w}, sa[4] = {ss.x, ss.y, ss.z, ss.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = low ? y[j] * ca[j] - p[j] * sa[j] : p[j] * sa[j] + y[j] * ca[j];
    } else {  // (2 i, 2 i + 1)
        const float2 cc = *reinterpret_cast<const float2 *>(c + (d >> 1)), ss = *reinterpret_cast<const float2 *>(s + (d >> 1));
        const float a = y[0], b = y[1], e = y[2], f = y[3];
        y[0] = a * cc.x - b * ss.x, y[1] = a * ss.x + b * cc.x;
        y[2] = e * cc.y - f * ss.y, y[3] = e * ss.y + f * cc.y;
    }
}

// scale of a block whose largest magnitude has these bits
__device__ __forceinline__ float block_scale(uint32_t amax)
{
    if (amax >= 0x7F800000u) return __uint_as_float(0x7FC00000u);
    const int k = max((int)(amax >> 23) - 127 - 8 + ((amax & 0x7FFFFFu) > 0x600000u), SCALE_FLOOR);
    return __uint_as_float((uint32_t)(k + 127) << 23);
}

// Blocks of threads [0, items * kvh * 2): one page's new tokens of one head, keys or values.  The rest: rotated queries.
// Item i of the sequence with items [row_start / page + 2 s, ..): a sequence of n rows touches (n - 2) / page + 2 pages at most.
template <typename T, int HD>
__global__ void __launch_bounds__(UPDATE_THREADS) paged_update_kernel(const Update u)
{
    smc_grid_dep_sync();
    const smc_paged_view &c = u.c;
    const int page = 1 << c.shift, tid = threadIdx.x;
    const long long jobs = (long long)u.items * c.kvh * 2;
    if (blockIdx.x >= jobs) {
        const long long at = (long long)(blockIdx.x - jobs) * UPDATE_THREADS + tid;
        const int per_row = u.heads * (HD / 4);
        const int r = (int)(at / per_row), e = (int)(at - (long long)r * per_row) * 4, d = e % HD;
        const int s = r < c.rows ? smc_paged_row_sequence(c, r) : -1;
        bool in = s >= 0;
        float y[4];
        if (in) {
            const smc_paged_seq sq = smc_paged_sequence(c, s);
            const int pos = sq.len - sq.n + r - sq.r0;
            in = pos >= 0 && pos < u.table_rows;
            if (!in && u.cosT) *u.status = SMC_STATUS_PAGED;
            const size_t row = (size_t)pos * (u.rope_dim >> 1);
            if (in) rotated4(static_cast<const T *>(u.q) + (long long)r * u.q_stride + (e - d), d, u.rope_dim, u.neox, u.cosT ? u.cosT + row : nullptr, u.sinT + row, y);
        }
        __syncwarp();  // in place: the two threads of a pair, both of one warp, have read it before either writes
        if (in) smc_paged_store4(static_cast<T *>(u.q_out) + (long long)r * u.heads * HD + e, y);
        return;
    }
    const int item = (int)(blockIdx.x / (2 * c.kvh)), rest = (int)(blockIdx.x - (unsigned)item * 2 * c.kvh), h = rest >> 1;
    const bool values = rest & 1;
    int s = item, local = 0;
    if (c.row_start) {  // the last s whose items start at or before this one
        int lo = 0, hi = c.batch;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if ((min(max(c.row_start[mid], 0), c.rows) >> c.shift) + 2 * mid <= item) lo = mid;
            else hi = mid;
        }
        s = lo, local = item - ((min(max(c.row_start[lo], 0), c.rows) >> c.shift) + 2 * lo);
    }
    const smc_paged_seq sq = smc_paged_sequence(c, s);
    const int p0 = sq.len - sq.n;
    if (sq.bad || p0 < 0 || (u.cosT && sq.len > u.table_rows)) {
        if (tid == 0) *u.status = SMC_STATUS_PAGED;
        return;
    }
    const int pg = (p0 >> c.shift) + local, start = pg << c.shift;
    if (sq.n == 0 || start >= sq.len || local < 0) return;
    const int id = smc_paged_page(c, s, pg);
    if (id < 0) {
        if (tid == 0) *u.status = SMC_STATUS_PAGED;
        return;
    }
    const int lo = max(p0 - start, 0), hi = min(sq.len - start, page);  // tokens [lo, hi) of the page are new
    const T *src = static_cast<const T *>(values ? u.v : u.k) + (long long)(sq.r0 + start - p0) * (values ? u.v_stride : u.k_stride) + (size_t)h * HD;
    const long long stride = values ? u.v_stride : u.k_stride;
    const size_t block = ((size_t)id * c.kvh + h) * ((size_t)HD << c.shift);
    uint8_t *dst = (values ? c.v : c.k) + block;
    float *scale = c.scales + ((size_t)id * c.kvh + h) * 2 + values;
    const bool rotate = !values && u.cosT;
    auto token4 = [&](int t, int d, float (&y)[4]) {
        const size_t row = (size_t)(start + t) * (u.rope_dim >> 1);
        rotated4(src + t * stride, d, u.rope_dim, u.neox, rotate ? u.cosT + row : nullptr, u.sinT + row, y);
    };
    constexpr int V = HD / 4;
    uint32_t amax = 0;
    for (int i = lo * V + tid; i < hi * V; i += UPDATE_THREADS) {
        float y[4];
        token4(i / V, i % V * 4, y);
#pragma unroll
        for (int j = 0; j < 4; ++j) amax = max(amax, __float_as_uint(y[j]) & 0x7FFFFFFFu);  // (as bits an undefined value is the largest)
    }
    __shared__ uint32_t part[UPDATE_THREADS / 32];
    amax = __reduce_max_sync(0xFFFFFFFFu, amax);
    if ((tid & 31) == 0) part[tid >> 5] = amax;
    const float old = lo > 0 ? *scale : 0.0f;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < UPDATE_THREADS / 32; ++i) amax = max(amax, part[i]);
    const float need = block_scale(amax);
    const float now = old != old || need != need ? __uint_as_float(0x7FC00000u) : fmaxf(old, need);
    const float inv = now == now ? 1.0f / now : 0.0f;
    if (tid == 0 && !(now == old)) *scale = now;
    if (lo > 0 && now > old) {  // the tokens that are there, under the new scale
        const float ratio = old * inv;
        if (values) {
            for (int i = tid; i < HD * lo; i += UPDATE_THREADS) {
                uint8_t *p = dst + ((size_t)(i / lo) << c.shift) + i % lo;
                float f[4];
                smc_e4m3x4_float(*p, f);
                f[0] *= ratio;
                *p = (uint8_t)smc_float_e4m3x4(f);
            }
        } else {
            for (int i = tid; i < V * lo; i += UPDATE_THREADS) {
                uint32_t *p = reinterpret_cast<uint32_t *>(dst) + i;
                float f[4];
                smc_e4m3x4_float(*p, f);
#pragma unroll
                for (int j = 0; j < 4; ++j) f[j] *= ratio;
                *p = smc_float_e4m3x4(f);
            }
        }
    }
    for (int i = lo * V + tid; i < hi * V; i += UPDATE_THREADS) {
        const int t = i / V, d = i % V * 4;
        float y[4];
        token4(t, d, y);
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = now == now ? y[j] * inv : 0.0f;
        const uint32_t w = smc_float_e4m3x4(y);
        if (!values) *reinterpret_cast<uint32_t *>(dst + (size_t)t * HD + d) = w;
        else
#pragma unroll
            for (int j = 0; j < 4; ++j) dst[((size_t)(d + j) << c.shift) + t] = (uint8_t)(w >> (8 * j));
    }
}

// One block of threads = one page and head.  K: four neighbours of a token a thread; V: sixteen tokens of a dimension.
template <typename T, int HD>
__global__ void __launch_bounds__(128) paged_read_kernel(const smc_paged_view c, const int *pages, int n, T *k, T *v, int *status)
{
    smc_grid_dep_sync();
    const int i = blockIdx.x / c.kvh, h = blockIdx.x % c.kvh, id = pages[i], page = 1 << c.shift;
    const bool there = id >= 0 && id < c.pages;
    if (!there && threadIdx.x == 0) *status = SMC_STATUS_PAGED;
    const size_t block = there ? (size_t)id * c.kvh + h : 0, stride = (size_t)c.kvh * HD, at = ((size_t)i << c.shift) * stride + (size_t)h * HD;
    const float sk = there ? c.scales[2 * block] : 0.0f, sv = there ? c.scales[2 * block + 1] : 0.0f;
    const uint8_t *pk = c.k + block * ((size_t)HD << c.shift), *pv = c.v + block * ((size_t)HD << c.shift);
    for (int j = threadIdx.x; j < (HD / 4) << c.shift; j += 128) {
        float f[4] = {};
        if (there) smc_e4m3x4_float(reinterpret_cast<const uint32_t *>(pk)[j], f);
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] *= sk;
        smc_paged_store4(k + at + (size_t)(j / (HD / 4)) * stride + j % (HD / 4) * 4, f);
    }
    for (int j = threadIdx.x; j < HD * (page / 16); j += 128) {
        const int d = j % HD, t0 = j / HD * 16;
        const uint4 raw = there ? *reinterpret_cast<const uint4 *>(pv + ((size_t)d << c.shift) + t0) : make_uint4(0, 0, 0, 0);
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float f[4];
            smc_e4m3x4_float(w[e], f);
#pragma unroll
            for (int b = 0; b < 4; ++b) v[at + (size_t)(t0 + 4 * e + b) * stride + d] = from_f<T>(f[b] * sv);
        }
    }
}

// The context's device for the length of a call.
struct OnDevice {
    int before = 0;
    bool moved = false;
    explicit OnDevice(int device)
    {
        if (cudaGetDevice(&before) == cudaSuccess && before != device) moved = cudaSetDevice(device) == cudaSuccess;
    }
    ~OnDevice()
    {
        if (moved) cudaSetDevice(before);
    }
};

bool aligned(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check_cache(smc_ctx *ctx, const char *who, const smc_paged_kv *kv, int dtype)
{
    if (!ctx || !kv || !kv->k || !kv->v || !kv->scales || kv->pages <= 0 || kv->kv_heads <= 0) return smc_fail(ctx, SMC_E_INVALID, "%s: bad cache", who);
    if (kv->page != 16 && kv->page != 32 && kv->page != 64) return smc_fail(ctx, SMC_E_UNSUPPORTED, "%s: pages of 16, 32 or 64 tokens, not %d", who, kv->page);
    if (kv->head_dim != 64 && kv->head_dim != 128) return smc_fail(ctx, SMC_E_UNSUPPORTED, "%s: heads of 64 or 128, not %d", who, kv->head_dim);
    if (kv->kv_heads > 65535) return smc_fail(ctx, SMC_E_UNSUPPORTED, "%s: %d key/value heads", who, kv->kv_heads);
    if (!aligned(kv->k) || !aligned(kv->v) || (reinterpret_cast<uintptr_t>(kv->scales) & 7)) return smc_fail(ctx, SMC_E_INVALID, "%s: cache pointers are not aligned to 16 bytes", who);
    if (dtype != SMC_F32 && dtype != SMC_BF16) return smc_fail(ctx, SMC_E_UNSUPPORTED, "%s: activations of type %d (fp32 and bfloat16 are served)", who, dtype);
    return SMC_OK;
}

int check_seqs(smc_ctx *ctx, const char *who, const smc_paged_seqs *sq)
{
    if (!sq || sq->batch < 0 || sq->rows < 0 || sq->width < 0) return smc_fail(ctx, SMC_E_INVALID, "%s: bad sequences", who);
    if (sq->batch > 0 && (!sq->lengths || (sq->width > 0 && !sq->table))) return smc_fail(ctx, SMC_E_INVALID, "%s: bad sequences", who);
    if (!sq->row_start && sq->rows != sq->batch) return smc_fail(ctx, SMC_E_INVALID, "%s: %d rows for %d sequences of one row", who, sq->rows, sq->batch);
    return SMC_OK;
}

bool bad_rows(const void *p, long long stride, int heads, int hd, int dtype)
{
    return !p || !aligned(p) || stride < (long long)heads * hd || stride * (dtype == SMC_F32 ? 4 : 2) % 16 != 0;
}

smc_paged_view view(const smc_paged_kv *kv, const smc_paged_seqs *sq)
{
    smc_paged_view c{};
    c.k = static_cast<uint8_t *>(kv->k), c.v = static_cast<uint8_t *>(kv->v), c.scales = kv->scales;
    c.pages = kv->pages, c.kvh = kv->kv_heads, c.shift = kv->page == 16 ? 4 : kv->page == 32 ? 5 : 6;
    if (sq) c.table = sq->table, c.lengths = sq->lengths, c.row_start = sq->row_start, c.batch = sq->batch, c.width = sq->width, c.rows = sq->rows;
    return c;
}

}  // namespace

int smc_paged_update_dev(smc_ctx *ctx, const smc_paged_kv *kv, const smc_paged_seqs *seqs, int dtype, const void *d_k, long long k_stride, const void *d_v,
                         long long v_stride, const void *d_q, long long q_stride, void *d_q_out, int heads, const float *d_cos, const float *d_sin, int rope_dim,
                         int table_rows, int neox, void *stream)
{
    int rc = check_cache(ctx, "paged_update", kv, dtype);
    if (!rc) rc = check_seqs(ctx, "paged_update", seqs);
    if (rc) return rc;
    if (seqs->rows == 0 || seqs->batch == 0) return SMC_OK;
    if (bad_rows(d_k, k_stride, kv->kv_heads, kv->head_dim, dtype) || bad_rows(d_v, v_stride, kv->kv_heads, kv->head_dim, dtype) ||
        (d_q && (heads <= 0 || !d_q_out || !aligned(d_q_out) || bad_rows(d_q, q_stride, heads, kv->head_dim, dtype))))
        return smc_fail(ctx, SMC_E_INVALID, "paged_update: rows must start on 16-byte boundaries and hold their heads");
    if (d_q && d_q == d_q_out && q_stride != (long long)heads * kv->head_dim) return smc_fail(ctx, SMC_E_INVALID, "paged_update: queries in place are contiguous rows");
    if ((d_cos == nullptr) != (d_sin == nullptr)) return smc_fail(ctx, SMC_E_INVALID, "paged_update: one of the rotation's tables is missing");
    if (d_cos && (rope_dim <= 0 || rope_dim > kv->head_dim || rope_dim % 8 || table_rows <= 0 || !aligned(d_cos) || !aligned(d_sin)))
        return smc_fail(ctx, SMC_E_INVALID, "paged_update: rotation of %d of %d dimensions, a multiple of 8, by tables of %d rows on 16-byte boundaries", rope_dim, kv->head_dim, table_rows);
    Update u{};
    u.c = view(kv, seqs), u.k = d_k, u.v = d_v, u.q = d_q, u.q_out = d_q_out, u.k_stride = k_stride, u.v_stride = v_stride, u.q_stride = q_stride;
    u.heads = d_q ? heads : 0, u.rope_dim = d_cos ? rope_dim : 0, u.table_rows = d_cos ? table_rows : 0x7FFFFFFF, u.neox = neox, u.cosT = d_cos, u.sinT = d_sin, u.status = ctx->d_status;
    const long long items = seqs->row_start ? (seqs->rows >> u.c.shift) + 2LL * seqs->batch : seqs->batch;
    const long long grid = items * kv->kv_heads * 2 + ((long long)seqs->rows * u.heads * (kv->head_dim / 4) + UPDATE_THREADS - 1) / UPDATE_THREADS;
    if (grid > 0x7FFFFFFF) return smc_fail(ctx, SMC_E_UNSUPPORTED, "paged_update: %lld rows and sequences in one call", (long long)seqs->rows + seqs->batch);
    u.items = (int)items;
    OnDevice on(ctx->device);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    auto go = [&](auto kernel) { smc_launch_dep(ctx->use_pdl, kernel, dim3((unsigned)grid), dim3(UPDATE_THREADS), 0, s, u); };
    if (dtype == SMC_F32) kv->head_dim == 128 ? go(paged_update_kernel<float, 128>) : go(paged_update_kernel<float, 64>);
    else kv->head_dim == 128 ? go(paged_update_kernel<bf16, 128>) : go(paged_update_kernel<bf16, 64>);
    SMC_LAUNCH_CHECK(ctx);
    return SMC_OK;
}

int smc_paged_read_dev(smc_ctx *ctx, const smc_paged_kv *kv, const int *d_pages, int n, int dtype, void *d_k, void *d_v, void *stream)
{
    const int rc = check_cache(ctx, "paged_read", kv, dtype);
    if (rc) return rc;
    if (n < 0 || (n > 0 && (!d_pages || !d_k || !d_v || !aligned(d_k) || !aligned(d_v)))) return smc_fail(ctx, SMC_E_INVALID, "paged_read: bad arguments");
    if (n == 0) return SMC_OK;
    if ((long long)n * kv->kv_heads > 0x7FFFFFFF) return smc_fail(ctx, SMC_E_UNSUPPORTED, "paged_read: %d pages in one call", n);
    OnDevice on(ctx->device);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    auto go = [&](auto kernel, auto *k, auto *v) {
        smc_launch_dep(ctx->use_pdl, kernel, dim3((unsigned)(n * kv->kv_heads)), dim3(128), 0, s, view(kv, nullptr), d_pages, n, k, v, ctx->d_status);
    };
    if (dtype == SMC_F32) kv->head_dim == 128 ? go(paged_read_kernel<float, 128>, (float *)d_k, (float *)d_v) : go(paged_read_kernel<float, 64>, (float *)d_k, (float *)d_v);
    else kv->head_dim == 128 ? go(paged_read_kernel<bf16, 128>, (bf16 *)d_k, (bf16 *)d_v) : go(paged_read_kernel<bf16, 64>, (bf16 *)d_k, (bf16 *)d_v);
    SMC_LAUNCH_CHECK(ctx);
    return SMC_OK;
}

int64_t smc_paged_attention_work(smc_ctx *ctx, const smc_paged_kv *kv, int batch, int rows, int heads, int max_rows, int max_len)
{
    if (check_cache(ctx, "paged_attention_work", kv, SMC_F32)) return -1;
    if (batch < 0 || rows < 0 || heads <= 0 || heads % kv->kv_heads || max_rows < 0 || max_len < 0) return smc_fail(ctx, -1, "paged_attention_work: bad arguments");
    // (the type of the activations is not known here: the form may be either)
    const int group = heads / kv->kv_heads;
    size_t n = 0;
    if (smc_paged_decode_takes(1, group, max_rows)) n = smc_paged_decode_work(ctx, kv->kv_heads, batch, heads, kv->head_dim, max_rows, max_len);
    if (!smc_paged_decode_takes(0, group, max_rows)) n = std::max(n, smc_paged_prompt_work(ctx, kv->kv_heads, batch, rows, heads, kv->head_dim, max_len));
    return (int64_t)n;
}

int smc_paged_attention_dev(smc_ctx *ctx, const smc_paged_kv *kv, const smc_paged_seqs *seqs, int dtype, const void *d_q, long long q_stride, void *d_out, int heads,
                            float scale, int window, int max_rows, int max_len, void *d_work, long long work_bytes, void *stream)
{
    int rc = check_cache(ctx, "paged_attention", kv, dtype);
    if (!rc) rc = check_seqs(ctx, "paged_attention", seqs);
    if (rc) return rc;
    if (heads <= 0 || heads % kv->kv_heads || window < 0 || max_rows < 0 || max_len < 0) return smc_fail(ctx, SMC_E_INVALID, "paged_attention: bad arguments");
    if (seqs->rows == 0 || seqs->batch == 0) return SMC_OK;
    if (bad_rows(d_q, q_stride, heads, kv->head_dim, dtype) || !d_out || !aligned(d_out))
        return smc_fail(ctx, SMC_E_INVALID, "paged_attention: rows must start on 16-byte boundaries and hold their heads");
    if ((long long)seqs->batch * kv->kv_heads * ((long long)seqs->width * kv->page / 64 + 1) > 0x7FFFFFFF)
        return smc_fail(ctx, SMC_E_UNSUPPORTED, "paged_attention: a table of %d x %d pages of %d heads", seqs->batch, seqs->width, kv->kv_heads);
    OnDevice on(ctx->device);
    const smc_paged_query q{d_q, q_stride, d_out, dtype == SMC_BF16, heads, kv->head_dim, window, max_rows, max_len, scale};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (max_rows == 0) return smc_fail(ctx, SMC_E_INVALID, "paged_attention: %d rows, none of a sequence", seqs->rows);
    const int64_t need = smc_paged_attention_work(ctx, kv, seqs->batch, seqs->rows, heads, max_rows, max_len);
    if (need > 0 && (!d_work || !aligned(d_work) || work_bytes < need))
        return smc_fail(ctx, SMC_E_INVALID, "paged_attention: %lld bytes of work space are not enough, or not on a 16-byte boundary", work_bytes);
    if (smc_paged_decode_takes(q.bf16, heads / kv->kv_heads, max_rows)) return smc_launch_paged_decode(ctx, view(kv, seqs), q, static_cast<float *>(d_work), s);
    return smc_launch_paged_prompt(ctx, view(kv, seqs), q, static_cast<float *>(d_work), s);
}
