// Rows of q, k and v into the paged 8-bit cache: q and k rotated at their positions, k and v of each page and head brought
// to one power-of-two scale and rounded once.
//
//   y[d] = x[d] cos[d] - x[d + D/2] sin[d],  y[d + D/2] = x[d + D/2] cos[d] + x[d] sin[d]      (q, k)
//   scale(page, head) = max(smallest 2^e, e >= -64, with max |y| <= top 2^e; the page's old scale if it held tokens before)
//   code = round(y / scale)
//
// Scales are powers of two because a page fills over many calls: where a later token needs a larger scale, the page's tokens are
// moved to it, and a power of two moves e4m3 codes without loss (but for the smallest) and costs int8 codes only the bits
// that fall off, at most one step of the final scale in all. The division by the scale is exact, and the two products of the rotation are added with
// rounding to odd, so a code is the correctly rounded one of the exact value.
//
// Bound by HBM: qkv is read once, q and the codes are written once. A block of the first kind owns one page of one sequence,
// one head and k or v: no other block writes that page's codes or scale, so nothing is atomic. Its threads keep the call's rows of the
// page in registers (64 values each) between the maximum and the rounding. A block of the second kind rotates q. 8192 rows of 32/8 heads of
// 128, fp16 to e4m3: 44.7 us, 4.2 TB/s (0.65 of what a copy moves), 33 us of them for q; 64 single rows: 3.4 us.
#include <climits>

#include "kv_cache.cuh"
#include "launch.cuh"

namespace macko {
namespace {

constexpr int kItems = 4;         // pairs of 8 dimensions, D/2 apart, that a thread of a page's block holds
constexpr int kQueryItems = 4;    // the same for a thread that rotates q

struct AppendArgs {
    CacheView cache;
    RowsView rows;
    const uint16_t *qkv;
    const __half *cos_table, *sin_table;
    uint16_t *q;
    long long row_stride;
    int heads, units, page_blocks;
    int query_items;   // of a thread that rotates q: 1 or kQueryItems
};

// Page `unit` of those that the call's rows fall on, in the order of the sequences: the rows on it and where they go.
struct PageRows {
    int sequence, first_row, count, position;   // rows [first_row, + count) at positions position, ...; count 0: no such page
};

// All threads of the block; two barriers per blockDim.x sequences.
__device__ PageRows find_page(const RowsView &r, int page_log2, int unit, int *shared)
{
    PageRows found = {0, 0, 0, 0};
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    if (r.start == nullptr) {
        const Sequence s = sequence_at(r, unit);
        if (s.begin() >= 0 && s.begin() < r.capacity) found = PageRows{unit, s.first, 1, s.begin()};
        return found;
    }
    int before = 0;
    for (int base = 0; base < r.sequences; base += blockDim.x) {
        int pages = 0, begin = 0, end = 0;
        Sequence s = {0, 0, 0};
        if (base + tid < r.sequences) {
            s = sequence_at(r, base + tid);
            begin = max(s.begin(), 0);
            end = min(s.length, r.capacity);
            if (begin < end) pages = ((end - 1) >> page_log2) - (begin >> page_log2) + 1;
        }
        int sum = pages;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
        if (lane == 31) shared[warp] = sum;
        __syncthreads();
        int total = 0;
        for (int w = 0; w < warps; ++w) {
            if (w < warp) sum += shared[w];
            total += shared[w];
        }
        const int lo = before + sum - pages;
        if (unit >= lo && unit < lo + pages) {
            const int page = (begin >> page_log2) + unit - lo;
            const int from = max(begin, page << page_log2), to = min(end, (page + 1) << page_log2);
            shared[32] = base + tid;
            shared[33] = s.first + from - s.begin();
            shared[34] = to - from;
            shared[35] = from;
        }
        before += total;
        __syncthreads();
        if (unit < before) return PageRows{shared[32], shared[33], shared[34], shared[35]};
    }
    return found;
}

// Rotates 8 dimensions of the first half of a head and their partners, to odd.
template <bool BF16>
__device__ __forceinline__ void rotate(const uint4 &lo, const uint4 &hi, const uint4 &cos8, const uint4 &sin8, float (&y)[16])
{
    const uint32_t *l = &lo.x, *h = &hi.x, *c = &cos8.x, *s = &sin8.x;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 a = unpack2<BF16>(l[j]), b = unpack2<BF16>(h[j]), co = unpack2<false>(c[j]), si = unpack2<false>(s[j]);
        y[2 * j] = difference_to_odd(a.x, co.x, b.x, si.x);
        y[2 * j + 1] = difference_to_odd(a.y, co.y, b.y, si.y);
        y[8 + 2 * j] = difference_to_odd(b.x, co.x, -a.x, si.x);
        y[8 + 2 * j + 1] = difference_to_odd(b.y, co.y, -a.y, si.y);
    }
}

// Smallest power of two s >= 2^-64 with |x| <= top * s, from the bits of the finite |x|; top = 127 = 1.984375 * 2^6 or 448 = 1.75 * 2^8.
template <bool E4M3>
__device__ __forceinline__ float scale_for(uint32_t magnitude)
{
    int e = (int)(magnitude >> 23) - (E4M3 ? 8 : 6);          // biased exponent of the scale for fractions up to the top's
    if ((magnitude & 0x7fffffu) > (E4M3 ? 0x600000u : 0x7e0000u)) ++e;
    return __uint_as_float((uint32_t)max(e, 127 - 64) << 23);
}

template <bool BF16, bool E4M3, int D>
__global__ void __launch_bounds__(512)
rope_append_kernel(const AppendArgs a)
{
    constexpr int kPerRow = D / 16;   // threads of a row
    __shared__ int found[36];
    __shared__ uint32_t largest[16];
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x;
    const RowsView &r = a.rows;
    const CacheView &c = a.cache;
    const int hq = a.heads, hkv = c.kv_heads;

    if ((int)blockIdx.x >= a.page_blocks) {
        // q: blocks over (row, head, part of the head). The sequence of the block's first row is looked for by all threads at once, in one
        // way to memory; the others' rows are nearly always its own.
        const long long base = (long long)((int)blockIdx.x - a.page_blocks) * blockDim.x * a.query_items / kPerRow;   // row and head
        const int row0 = (int)(base / hq), head0 = (int)(base % hq);
        int behind = r.rows;   // rows from here on belong to no sequence
        if (r.start != nullptr) {
            behind = r.sequences > 0 ? __ldcg(r.start + r.sequences) : 0;
            if (tid == 0) found[0] = r.sequences;
            __syncthreads();
            for (int i = tid; i < r.sequences; i += blockDim.x) {
                const Sequence s = sequence_at(r, i);
                if (row0 >= s.first && row0 < s.first + s.count) {
                    found[0] = i;
                    found[1] = s.first;
                    found[2] = s.count;
                    found[3] = s.length;
                }
            }
            __syncthreads();
        }
        uint4 lo[kQueryItems], hi[kQueryItems], co[kQueryItems], si[kQueryItems];
        long long to[kQueryItems];   // in q, or -1
#pragma unroll
        for (int i = 0; i < kQueryItems; ++i) {
            if (i >= a.query_items) break;
            const int item = i * (int)blockDim.x + tid, part = item % kPerRow, row_head = head0 + item / kPerRow;
            const int row = row0 + row_head / hq, head = row_head % hq;
            int position = -1;
            if (row < min(r.rows, behind)) {
                Sequence s = {0, 0, 0};
                if (r.start == nullptr) {
                    s = sequence_at(r, row);
                } else {
                    int seq = found[0];
                    if (seq < r.sequences) s = Sequence{found[1], found[2], found[3]};
                    else seq = -1;
                    while (row >= s.first + s.count && ++seq < r.sequences) s = sequence_at(r, seq);
                }
                if (row >= s.first && row < s.first + s.count) position = s.begin() + row - s.first;
            }
            const bool there = position >= 0 && position < r.capacity;
            to[i] = row < r.rows ? ((long long)row * hq + head) * D + 8 * part : -1;
            const uint16_t *x = a.qkv + (long long)row * a.row_stride + head * D + 8 * part;
            const long long at = (long long)position * D + 8 * part;
            load_if(lo[i], x, there);
            load_if(hi[i], x + D / 2, there);
            load_if(co[i], a.cos_table + at, there);
            load_if(si[i], a.sin_table + at, there);
        }
#pragma unroll
        for (int i = 0; i < kQueryItems; ++i) {
            if (i >= a.query_items) break;
            float y[16];
            rotate<BF16>(lo[i], hi[i], co[i], si[i], y);
            if (to[i] < 0) continue;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                (&lo[i].x)[j] = pack2<BF16>(y[2 * j], y[2 * j + 1]);
                (&hi[i].x)[j] = pack2<BF16>(y[8 + 2 * j], y[8 + 2 * j + 1]);
            }
            *reinterpret_cast<uint4 *>(a.q + to[i]) = lo[i];
            *reinterpret_cast<uint4 *>(a.q + to[i] + D / 2) = hi[i];
        }
        return;
    }

    const bool is_v = blockIdx.x & 1u;
    const int head = (int)((blockIdx.x >> 1) % (unsigned)hkv), unit = (int)((blockIdx.x >> 1) / (unsigned)hkv);
    const PageRows rows = find_page(r, c.page_log2, unit, found);
    if (rows.count == 0) return;
    const int page = page_at(c, r, rows.sequence, rows.position);
    if (page < 0) return;
    const int slot = rows.position & ((1 << c.page_log2) - 1);
    uint8_t *codes = (is_v ? c.v + (long long)page * c.v_stride : c.k + (long long)page * c.k_stride) + ((long long)head << c.page_log2) * D;
    float *scale = is_v ? c.v_scale + (long long)page * c.v_scale_stride + head : c.k_scale + (long long)page * c.k_scale_stride + head;
    const float old = slot > 0 ? __ldcg(scale) : 0.f;

    const int rows_apart = (int)blockDim.x / kPerRow;   // between a thread's items
    uint4 lo[kItems], hi[kItems], co[kItems], si[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        if (i * rows_apart >= rows.count) break;
        const int item = i * (int)blockDim.x + tid, row = item / kPerRow, part = item % kPerRow;
        const bool there = row < rows.count;
        const uint16_t *x = a.qkv + (long long)(rows.first_row + row) * a.row_stride + (hq + (is_v ? hkv : 0) + head) * D + 8 * part;
        const long long at = (long long)(rows.position + row) * D + 8 * part;
        load_if(lo[i], x, there);
        load_if(hi[i], x + D / 2, there);
        load_if(co[i], a.cos_table + at, there && !is_v);
        load_if(si[i], a.sin_table + at, there && !is_v);
    }
    float y[kItems][16];
    uint32_t most = 0u;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        if (i * rows_apart >= rows.count) break;
        if (is_v) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 l = unpack2<BF16>((&lo[i].x)[j]), h = unpack2<BF16>((&hi[i].x)[j]);
                y[i][2 * j] = l.x;
                y[i][2 * j + 1] = l.y;
                y[i][8 + 2 * j] = h.x;
                y[i][8 + 2 * j + 1] = h.y;
            }
        } else {
            rotate<BF16>(lo[i], hi[i], co[i], si[i], y[i]);
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) most = max(most, __float_as_uint(y[i][j]) & 0x7fffffffu);
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if ((tid & 31) == 0) largest[tid >> 5] = most;
    __syncthreads();   // every thread has read the old scale as well
    for (int w = 0; w < (int)blockDim.x >> 5; ++w) most = max(most, largest[w]);

    const uint32_t infinite = 0x7f800000u;
    const bool finite = most < infinite && (__float_as_uint(old) & 0x7fffffffu) < infinite;
    const float now = finite ? fmaxf(scale_for<E4M3>(most), old) : __uint_as_float(0x7fffffffu);
    if (tid == 0) *scale = now;
    if (finite && slot > 0 && now != old) {
        const float factor = old / now;
        for (int i = tid; i < slot * (D / 16); i += blockDim.x) {
            uint4 *at = reinterpret_cast<uint4 *>(codes) + i;
            uint4 x = *at;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t lo, hi;
                codes_to_half<E4M3>((&x.x)[j], lo, hi);
                const float2 l = unpack2<false>(lo), h = unpack2<false>(hi);
                (&x.x)[j] = codes_from_float<E4M3>(l.x * factor, l.y * factor, h.x * factor, h.y * factor);
            }
            *at = x;
        }
    }
    const float inverse = finite ? 1.f / now : 0.f;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        if (i * rows_apart >= rows.count) break;
        const int item = i * (int)blockDim.x + tid, row = item / kPerRow, part = item % kPerRow;
        if (row < rows.count) {
            uint2 out[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float *v = y[i] + 8 * h;
                out[h].x = codes_from_float<E4M3>(v[0] * inverse, v[1] * inverse, v[2] * inverse, v[3] * inverse);
                out[h].y = codes_from_float<E4M3>(v[4] * inverse, v[5] * inverse, v[6] * inverse, v[7] * inverse);
            }
            uint8_t *to = codes + (long long)(slot + row) * D + 8 * part;
            *reinterpret_cast<uint2 *>(to) = finite ? out[0] : make_uint2(0u, 0u);
            *reinterpret_cast<uint2 *>(to + D / 2) = finite ? out[1] : make_uint2(0u, 0u);
        }
    }
}

template <bool BF16, bool E4M3>
int launch_append(const AppendArgs &a, int threads, unsigned blocks, cudaStream_t stream)
{
    switch (a.cache.head_dim) {
    case 64: return launch_pdl("rope_append", rope_append_kernel<BF16, E4M3, 64>, dim3(blocks), dim3(threads), 1, 0, stream, a);
    case 128: return launch_pdl("rope_append", rope_append_kernel<BF16, E4M3, 128>, dim3(blocks), dim3(threads), 1, 0, stream, a);
    default: return launch_pdl("rope_append", rope_append_kernel<BF16, E4M3, 256>, dim3(blocks), dim3(threads), 1, 0, stream, a);
    }
}

}  // namespace

int check_cache(const char *what, const macko_kv_cache *c, CacheView *view)
{
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) return fail(MACKO_ERR_INVALID_ARGUMENT, "%s: the cache has a null pointer", what);
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
        return fail(MACKO_ERR_INVALID_ARGUMENT, "%s: page_size %d (16, 32, 64 and 128 are built)", what, c->page_size);
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return fail(MACKO_ERR_INVALID_ARGUMENT, "%s: head_dim %d (64, 128 and 256 are built)", what, c->head_dim);
    if (c->code != MACKO_KV_INT8 && c->code != MACKO_KV_E4M3) return fail(MACKO_ERR_INVALID_ARGUMENT, "%s: unknown code %d", what, c->code);
    if (c->pages <= 0 || c->kv_heads <= 0) return fail(MACKO_ERR_INVALID_ARGUMENT, "%s: pages=%lld kv_heads=%d", what, (long long)c->pages, c->kv_heads);
    if (c->pages > INT_MAX || c->kv_heads > 4096) return fail(MACKO_ERR_SIZE_OVERFLOW, "%s: pages=%lld kv_heads=%d", what, (long long)c->pages, c->kv_heads);
    const int64_t page_bytes = (int64_t)c->kv_heads * c->page_size * c->head_dim;
    if (c->k_page_stride < page_bytes || c->v_page_stride < page_bytes || c->k_scale_stride < c->kv_heads || c->v_scale_stride < c->kv_heads)
        return fail(MACKO_ERR_INVALID_ARGUMENT, "%s: a page stride is smaller than a page", what);
    if (c->k_page_stride > (1ll << 36) / c->pages || c->v_page_stride > (1ll << 36) / c->pages || c->k_scale_stride > (1ll << 40) || c->v_scale_stride > (1ll << 40))
        return fail(MACKO_ERR_SIZE_OVERFLOW, "%s: keys or values of more than 2^36 bytes", what);   // 32 bits count them by 16
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || c->k_page_stride % 16 || c->v_page_stride % 16 || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4))
        return fail(MACKO_ERR_MISALIGNED, "%s: codes and the strides of their pages must be multiples of 16 bytes, scales of 4", what);
    int log2 = 4;
    while ((1 << log2) < c->page_size) ++log2;
    *view = CacheView{static_cast<uint8_t *>(c->k), static_cast<uint8_t *>(c->v), c->k_scale, c->v_scale, c->k_page_stride, c->v_page_stride,
                      c->k_scale_stride, c->v_scale_stride, (int)c->pages, c->kv_heads, log2, c->head_dim};
    return MACKO_OK;
}

int check_rows(const char *what, const macko_kv_rows *r, int page_size, RowsView *view)
{
    if (!r || r->sequences < 0 || r->rows < 0 || r->table_width < 0)
        return fail(MACKO_ERR_INVALID_ARGUMENT, "%s: null or negative batch", what);
    if (r->sequences > 1 << 20 || r->rows > 1 << 24 || r->table_width * page_size > INT_MAX - (1 << 24))
        return fail(MACKO_ERR_SIZE_OVERFLOW, "%s: sequences=%lld rows=%lld table_width=%lld", what, (long long)r->sequences, (long long)r->rows,
                    (long long)r->table_width);
    if (r->sequences > 0 && (!r->lengths || (r->table_width > 0 && !r->page_table)))
        return fail(MACKO_ERR_INVALID_ARGUMENT, "%s: null page_table or lengths", what);
    if (r->sequences > 1 && r->table_stride < r->table_width) return fail(MACKO_ERR_INVALID_ARGUMENT, "%s: table_stride smaller than table_width", what);
    if (!r->query_start && r->rows != r->sequences)
        return fail(MACKO_ERR_INVALID_ARGUMENT, "%s: %lld rows for %lld sequences without query_start", what, (long long)r->rows, (long long)r->sequences);
    if (!aligned(r->page_table, 4) || !aligned(r->lengths, 4) || !aligned(r->query_start, 4))
        return fail(MACKO_ERR_MISALIGNED, "%s: page_table, lengths and query_start must be 4-byte aligned", what);
    *view = RowsView{r->page_table, r->lengths, r->query_start, r->table_stride, (int)r->table_width, (int)(r->table_width * page_size),
                     (int)r->sequences, (int)r->rows};
    return MACKO_OK;
}

}  // namespace macko

using namespace macko;

extern "C" int macko_cache_rope_append(const macko_kv_cache *cache, const macko_kv_rows *batch, const void *qkv, int64_t row_stride,
                                       int32_t type, const void *cos_table, const void *sin_table, void *q, int32_t heads, void *stream)
{
    AppendArgs a = {};
    if (int st = check_cache("rope_append", cache, &a.cache)) return st;
    if (int st = check_rows("rope_append", batch, cache->page_size, &a.rows)) return st;
    if (heads <= 0 || heads > 4096 || heads % cache->kv_heads)
        return fail(MACKO_ERR_INVALID_ARGUMENT, "rope_append: %d heads for %d key heads", heads, cache->kv_heads);
    if (type != MACKO_FP16 && type != MACKO_BF16) return fail(MACKO_ERR_INVALID_ARGUMENT, "rope_append: unknown type %d", type);
    if (a.rows.rows == 0) return MACKO_OK;
    if (!qkv || !q || !cos_table || !sin_table) return fail(MACKO_ERR_INVALID_ARGUMENT, "rope_append: null pointer");
    if (row_stride < (int64_t)(heads + 2 * cache->kv_heads) * cache->head_dim)
        return fail(MACKO_ERR_INVALID_ARGUMENT, "rope_append: row_stride %lld is smaller than a row", (long long)row_stride);
    if (!aligned(qkv, 16) || !aligned(q, 16) || !aligned(cos_table, 16) || !aligned(sin_table, 16) || row_stride % 8)
        return fail(MACKO_ERR_MISALIGNED, "rope_append: rows, q and the tables must be 16-byte aligned");
    a.qkv = static_cast<const uint16_t *>(qkv);
    a.cos_table = static_cast<const __half *>(cos_table);
    a.sin_table = static_cast<const __half *>(sin_table);
    a.q = static_cast<uint16_t *>(q);
    a.row_stride = row_stride;
    a.heads = heads;
    // a page's rows in registers, 64 values a thread; a sequence of n rows touches at most n pages and at most n / page_size + 2
    const int page = cache->page_size, d = cache->head_dim;
    const int threads = page * d / 64 > 64 ? page * d / 64 : 64;
    const int64_t pages = a.rows.rows / page + 2 * (int64_t)a.rows.sequences;
    a.units = (int)(a.rows.rows < pages ? a.rows.rows : pages);
    const int64_t page_blocks = a.rows.sequences > 0 ? (int64_t)a.units * cache->kv_heads * 2 : 0;
    // one item a thread where all of them fit the GPU at once (64 rows of 32 + 8 heads of 128: 3.4 us for the whole call),
    // else four items a thread, whose loads are under way together (8192 rows: 46 us, 54 with two)
    a.query_items = (int64_t)a.rows.rows * heads * (d / 16) <= 148 * 1024 ? 1 : kQueryItems;
    const int64_t per_block = (int64_t)threads * a.query_items;
    const int64_t q_blocks = ((int64_t)a.rows.rows * heads * (d / 16) + per_block - 1) / per_block;   // per_block: whole heads
    if (page_blocks + q_blocks > INT_MAX)
        return fail(MACKO_ERR_SIZE_OVERFLOW, "rope_append: rows=%d heads=%d need too many blocks", a.rows.rows, heads);
    a.page_blocks = (int)page_blocks;
    const unsigned blocks = (unsigned)(page_blocks + q_blocks);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool e4m3 = cache->code == MACKO_KV_E4M3;
    if (type == MACKO_BF16) return e4m3 ? launch_append<true, true>(a, threads, blocks, s) : launch_append<true, false>(a, threads, blocks, s);
    return e4m3 ? launch_append<false, true>(a, threads, blocks, s) : launch_append<false, false>(a, threads, blocks, s);
}
