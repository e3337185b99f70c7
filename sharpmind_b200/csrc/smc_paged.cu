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

// Eight elements of a head, by unit 0 .. HD / 8 - 1: those of pairs (i, i + rope_dim / 2) in two fours where there is a rotation of that kind, neighbours
// otherwise.  `second` is where the second four are.
__device__ __forceinline__ void unit_place(int unit, int rope_dim, bool neox, int &first, int &second)
{
    const int half = rope_dim >> 1;
    if (neox && 4 * unit < half) first = 4 * unit, second = first + half;
    else first = neox ? rope_dim + 2 * (4 * unit - half) : 8 * unit, second = first + 4;
}
// a[], b[]: the unit's elements, rotated by the position's rows of the tables; every product and sum is rounded
__device__ __forceinline__ void unit_rotate(float (&a)[4], float (&b)[4], int first, int rope_dim, bool neox, const float *c, const float *s)
{
    if (first >= rope_dim) return;
    if (neox) {
        const float4 cc = *reinterpret_cast<const float4 *>(c + first), ss = *reinterpret_cast<const float4 *>(s + first);
        const float ca[4] = {cc.x, cc.y, cc.z, cc.w}, sa[4] = {ss.x, ss.y, ss.z, ss.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float x = a[j], y = b[j];
            a[j] = x * ca[j] - y * sa[j], b[j] = x * sa[j] + y * ca[j];
        }
    } else {
        const float4 cc = *reinterpret_cast<const float4 *>(c + (first >> 1)), ss = *reinterpret_cast<const float4 *>(s + (first >> 1));
        const float ca[4] = {cc.x, cc.y, cc.z, cc.w}, sa[4] = {ss.x, ss.y, ss.z, ss.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float *p = j < 2 ? a + 2 * j : b + 2 * (j - 2);
            const float x = p[0], y = p[1];
            p[0] = x * ca[j] - y * sa[j], p[1] = x * sa[j] + y * ca[j];
        }
    }
}

// scale of a block whose largest magnitude has these bits
__device__ __forceinline__ float block_scale(uint32_t amax)
{
    if (amax >= 0x7F800000u) return __uint_as_float(0x7FC00000u);
    const int k = max((int)(amax >> 23) - 127 - 8 + ((amax & 0x7FFFFFu) > 0x600000u), SCALE_FLOOR);
    return __uint_as_float((uint32_t)(k + 127) << 23);
}

// Blocks of threads [0, items * kvh * 2): one page's new tokens of one head, keys or values.  The rest: rotated queries, one row each.
// Item i of the sequence with items [row_start / page + 2 s, ..): a sequence of n rows touches (n - 2) / page + 2 pages at most.
// New values pass once through registers: their largest magnitude first, then, with the block's scale, their codes.  Keys: a thread takes units of
// eight elements of a token; values, which lie with a dimension's tokens side by side: a dimension of up to PER_V tokens.
// HBM is the bound: 4085 fp32 rows of 32 + 2 x 8 heads of 128, 176 MB, in 41 us from cold caches, 4.3 TB/s, 65 % of a copy's rate; 64 rows in bf16 12 us, one 5.4: latency.
template <typename T, int HD>
__global__ void __launch_bounds__(UPDATE_THREADS) paged_update_kernel(const Update u)
{
    constexpr int UNITS = HD / 8, PER_K = 64 * UNITS / UPDATE_THREADS, GROUPS_V = UPDATE_THREADS / HD, PER_V = 64 / GROUPS_V;
    smc_grid_dep_sync();
    const smc_paged_view &c = u.c;
    const int page = 1 << c.shift, tid = threadIdx.x;
    const long long jobs = (long long)u.items * c.kvh * 2;
    if (blockIdx.x >= jobs) {
        const int r = (int)(blockIdx.x - jobs), s = smc_paged_row_sequence(c, r);
        if (s < 0) return;
        const smc_paged_seq sq = smc_paged_sequence(c, s);
        const bool empty = sq.len == 0 && !sq.bad;  // an empty slot's queries go through as they are
        const int pos = empty ? 0 : sq.len - sq.n + r - sq.r0, rope_dim = empty ? 0 : u.rope_dim;
        if (pos < 0 || pos >= u.table_rows) {
            if (u.cosT && tid == 0) *u.status = SMC_STATUS_PAGED;
            return;
        }
        const float *cs = u.cosT + (size_t)pos * (rope_dim >> 1), *sn = u.sinT + (size_t)pos * (rope_dim >> 1);
        const T *src = static_cast<const T *>(u.q) + (long long)r * u.q_stride;
        T *dst = static_cast<T *>(u.q_out) + (long long)r * u.heads * HD;
#pragma unroll 2
        for (int i = tid; i < u.heads * UNITS; i += UPDATE_THREADS) {  // (in place: a unit is read and written by one thread)
            const int h = i / UNITS;
            int first, second;
            unit_place(i % UNITS, rope_dim, u.neox, first, second);
            float a[4], b[4];
            smc_paged_load4(src + h * HD + first, a), smc_paged_load4(src + h * HD + second, b);
            unit_rotate(a, b, first, rope_dim, u.neox, cs, sn);
            smc_paged_store4(dst + h * HD + first, a), smc_paged_store4(dst + h * HD + second, b);
        }
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
    if (sq.len == 0 && !sq.bad) return;
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
    const long long stride = values ? u.v_stride : u.k_stride;
    const T *src = static_cast<const T *>(values ? u.v : u.k) + (long long)(sq.r0 + start - p0) * stride + (size_t)h * HD;  // of token 0
    uint8_t *dst = (values ? c.v : c.k) + ((size_t)id * c.kvh + h) * ((size_t)HD << c.shift);
    float *scale = c.scales + ((size_t)id * c.kvh + h) * 2 + values;
    const float old = lo > 0 ? *scale : 0.0f;

    // ---- the new values and their largest magnitude
    static_assert(PER_K * 8 == PER_V, "");
    float x[PER_V];
    const int d = tid % HD, t0 = tid / HD * (page / GROUPS_V), t1 = t0 + page / GROUPS_V;  // values: tokens [t0, t1) of dimension d
    uint32_t amax = 0;
    if (values) {
#pragma unroll
        for (int i = 0; i < PER_V; ++i) {
            const int t = t0 + i;
            x[i] = t < t1 && t >= lo && t < hi ? to_f(src[t * stride + d]) : 0.0f;
        }
    } else {
#pragma unroll
        for (int i = 0; i < PER_K; ++i) {
            const int at = tid + i * UPDATE_THREADS, t = lo + at / UNITS;
            int first, second;
            unit_place(at % UNITS, u.rope_dim, u.neox, first, second);
            float a[4] = {}, b[4] = {};
            if (t < hi) {
                smc_paged_load4(src + t * stride + first, a), smc_paged_load4(src + t * stride + second, b);
                if (u.cosT) {
                    const size_t row = (size_t)(start + t) * (u.rope_dim >> 1);
                    unit_rotate(a, b, first, u.rope_dim, u.neox, u.cosT + row, u.sinT + row);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) x[8 * i + j] = a[j], x[8 * i + 4 + j] = b[j];
        }
    }
#pragma unroll
    for (int i = 0; i < PER_V; ++i) amax = max(amax, __float_as_uint(x[i]) & 0x7FFFFFFFu);  // (as bits an undefined value is the largest)
    __shared__ uint32_t part[UPDATE_THREADS / 32];
    amax = __reduce_max_sync(0xFFFFFFFFu, amax);
    if ((tid & 31) == 0) part[tid >> 5] = amax;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < UPDATE_THREADS / 32; ++i) amax = max(amax, part[i]);
    const float need = block_scale(amax);
    const float now = old != old || need != need ? __uint_as_float(0x7FC00000u) : fmaxf(old, need);
    const float inv = now == now ? 1.0f / now : 0.0f;
    if (tid == 0 && !(now == old)) *scale = now;

    // ---- tokens that are there, under the new scale
    if (lo > 0 && now > old) {
        const float ratio = old * inv;
        auto again = [&](uint32_t w) {
            float f[4];
            smc_e4m3x4_float(w, f);
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j] *= ratio;
            return smc_float_e4m3x4(f);
        };
        if (values) {
            for (int t = t0; t < min(t1, lo); t += 4) {
                uint32_t *p = reinterpret_cast<uint32_t *>(dst + ((size_t)d << c.shift) + t);
                const uint32_t was = *p, keep = t + 4 <= lo ? 0u : ~0u << (8 * (lo - t));  // bytes behind lo stay as they are
                *p = (again(was) & ~keep) | (was & keep);
            }
        } else {
            for (int i = tid; i < HD / 4 * lo; i += UPDATE_THREADS) reinterpret_cast<uint32_t *>(dst)[i] = again(reinterpret_cast<uint32_t *>(dst)[i]);
        }
    }
    // ---- codes of the new ones
#pragma unroll
    for (int i = 0; i < PER_V; ++i) x[i] = now == now ? x[i] * inv : 0.0f;
    if (values) {
        uint8_t *row = dst + ((size_t)d << c.shift) + t0;
#pragma unroll
        for (int i = 0; i < PER_V; i += 4) {
            const int t = t0 + i;
            if (t >= t1 || t + 4 <= lo || t >= hi) continue;
            const uint32_t w = smc_float_e4m3x4(*reinterpret_cast<const float(*)[4]>(x + i));
            if (t >= lo && t + 4 <= hi) *reinterpret_cast<uint32_t *>(row + i) = w;
            else
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (t + j >= lo && t + j < hi) row[i + j] = (uint8_t)(w >> (8 * j));
        }
    } else {
#pragma unroll
        for (int i = 0; i < PER_K; ++i) {
            const int at = tid + i * UPDATE_THREADS, t = lo + at / UNITS;
            if (t >= hi) continue;
            int first, second;
            unit_place(at % UNITS, u.rope_dim, u.neox, first, second);
            *reinterpret_cast<uint32_t *>(dst + (size_t)t * HD + first) = smc_float_e4m3x4(*reinterpret_cast<const float(*)[4]>(x + 8 * i));
            *reinterpret_cast<uint32_t *>(dst + (size_t)t * HD + second) = smc_float_e4m3x4(*reinterpret_cast<const float(*)[4]>(x + 8 * i + 4));
        }
    }
}

// One block of threads = one page and head.  K: eight neighbours of a token a thread; V: sixteen tokens of two dimensions.  All codes are on their way before the
// first is written.  HBM is the bound: 474 MB of codes and bf16 values in 84 us, 5.6 TB/s, 86 % of a copy's rate; 2000 tokens as fp32 6.8 us: latency.
template <typename T, int HD>
__global__ void __launch_bounds__(128) paged_read_kernel(const smc_paged_view c, const int *pages, int n, T *k, T *v, int *status)
{
    constexpr int PER_K = 64 * HD / 8 / 128, PER_V = 4 * (HD / 2) / 128;
    static_assert(PER_K >= 1 && PER_V >= 1, "");
    smc_grid_dep_sync();
    const int i = blockIdx.x / c.kvh, h = blockIdx.x % c.kvh, id = pages[i], page = 1 << c.shift, tid = threadIdx.x;
    const bool there = id >= 0 && id < c.pages;
    if (!there && tid == 0) *status = SMC_STATUS_PAGED;
    const size_t block = there ? (size_t)id * c.kvh + h : 0, stride = (size_t)c.kvh * HD, at = ((size_t)i << c.shift) * stride + (size_t)h * HD;
    const float2 scale = there ? *reinterpret_cast<const float2 *>(c.scales + 2 * block) : make_float2(0.0f, 0.0f);
    const uint8_t *pk = c.k + block * ((size_t)HD << c.shift), *pv = c.v + block * ((size_t)HD << c.shift);
    uint2 rk[PER_K];
    uint4 rv[PER_V][2];
#pragma unroll
    for (int e = 0; e < PER_K; ++e) {
        const int j = tid + 128 * e;
        rk[e] = there && j < (HD / 8) << c.shift ? *reinterpret_cast<const uint2 *>(pk + 8 * j) : make_uint2(0, 0);
    }
#pragma unroll
    for (int e = 0; e < PER_V; ++e) {
        const int j = tid + 128 * e, d = j % (HD / 2) * 2, t0 = j / (HD / 2) * 16;
        const bool in = there && t0 < page;
        rv[e][0] = in ? *reinterpret_cast<const uint4 *>(pv + ((size_t)d << c.shift) + t0) : make_uint4(0, 0, 0, 0);
        rv[e][1] = in ? *reinterpret_cast<const uint4 *>(pv + ((size_t)(d + 1) << c.shift) + t0) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int e = 0; e < PER_K; ++e) {
        const int j = tid + 128 * e;
        if (j >= (HD / 8) << c.shift) break;
        float f[8];
        smc_e4m3x4_float(rk[e].x, *reinterpret_cast<float(*)[4]>(f)), smc_e4m3x4_float(rk[e].y, *reinterpret_cast<float(*)[4]>(f + 4));
#pragma unroll
        for (int b = 0; b < 8; ++b) f[b] *= scale.x;
        T *dst = k + at + (size_t)(j / (HD / 8)) * stride + j % (HD / 8) * 8;
        if constexpr (sizeof(T) == 2) *reinterpret_cast<uint4 *>(dst) = make_uint4(pack2(f[0], f[1]), pack2(f[2], f[3]), pack2(f[4], f[5]), pack2(f[6], f[7]));
        else smc_paged_store4(dst, *reinterpret_cast<float(*)[4]>(f)), smc_paged_store4(dst + 4, *reinterpret_cast<float(*)[4]>(f + 4));
    }
#pragma unroll
    for (int e = 0; e < PER_V; ++e) {
        const int j = tid + 128 * e, d = j % (HD / 2) * 2, t0 = j / (HD / 2) * 16;
        if (t0 >= page) break;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            float a[4], b[4];
            smc_e4m3x4_float(w == 0 ? rv[e][0].x : w == 1 ? rv[e][0].y : w == 2 ? rv[e][0].z : rv[e][0].w, a);
            smc_e4m3x4_float(w == 0 ? rv[e][1].x : w == 1 ? rv[e][1].y : w == 2 ? rv[e][1].z : rv[e][1].w, b);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                T *dst = v + at + (size_t)(t0 + 4 * w + t) * stride + d;
                if constexpr (sizeof(T) == 2) *reinterpret_cast<uint32_t *>(dst) = pack2(a[t] * scale.y, b[t] * scale.y);
                else *reinterpret_cast<float2 *>(dst) = make_float2(a[t] * scale.y, b[t] * scale.y);
            }
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
    const long long grid = items * kv->kv_heads * 2 + (d_q ? seqs->rows : 0);
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
    const int group = heads / kv->kv_heads;
    return (int64_t)(smc_paged_decode_takes(group, max_rows, max_len) ? smc_paged_decode_work(ctx, kv->kv_heads, batch, heads, kv->head_dim, max_rows, max_len)
                                                             : smc_paged_prompt_work(ctx, kv->kv_heads, batch, rows, heads, kv->head_dim, max_len));
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
    if (smc_paged_decode_takes(heads / kv->kv_heads, max_rows, max_len)) return smc_launch_paged_decode(ctx, view(kv, seqs), q, static_cast<float *>(d_work), s);
    return smc_launch_paged_prompt(ctx, view(kv, seqs), q, static_cast<float *>(d_work), s);
}
