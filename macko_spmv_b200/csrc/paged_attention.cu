// Attention over the paged 8-bit cache.
#include <climits>

#include "kv_cache.cuh"
#include "launch.cuh"

namespace macko {
namespace {

struct AttentionArgs {
    CacheView cache;
    RowsView rows;
    const uint16_t *q;
    uint16_t *out;
    long long q_row_stride, q_head_stride;
    int heads;
    float scale;
};

// One warp per row and head: lane l holds dimensions l * D / 32 ..., tokens one after another with a running maximum.
template <bool BF16, bool E4M3, int D>
__global__ void __launch_bounds__(128)
attention_kernel(const AttentionArgs a)
{
    constexpr int V = D / 32;   // dimensions of a lane: 2, 4 or 8
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const RowsView &r = a.rows;
    const CacheView &c = a.cache;
    const int lane = threadIdx.x & 31;
    const long long id = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (id >= (long long)r.rows * a.heads) return;
    const int row = (int)(id / a.heads), head = (int)(id % a.heads), kv_head = head / (a.heads / c.kv_heads);
    int seq = row;
    if (r.start != nullptr) {
        seq = 0;
        for (int i = 1 + lane; i <= r.sequences; i += 32) seq += __ldg(r.start + i) <= row;
        seq = __reduce_add_sync(0xffffffffu, seq);
    }
    int seen = 0;
    if (seq < r.sequences) {
        const Sequence s = sequence_at(r, seq);
        if (row >= s.first && row < s.first + s.count) seen = max(0, min(s.begin() + row - s.first + 1, r.capacity));
    }
    float q[V], acc[V];
#pragma unroll
    for (int j = 0; j < V; j += 2) {
        const float2 t = unpack2<BF16>(*reinterpret_cast<const uint32_t *>(a.q + row * a.q_row_stride + head * a.q_head_stride + lane * V + j));
        q[j] = t.x * a.scale;
        q[j + 1] = t.y * a.scale;
        acc[j] = acc[j + 1] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int t = 0; t < seen; ++t) {
        const int page = page_at(c, r, seq, t);
        if (page < 0) continue;
        const long long at = (((long long)kv_head << c.page_log2) + (t & ((1 << c.page_log2) - 1))) * D + lane * V;
        const uint8_t *kp = c.k + page * c.k_stride + at, *vp = c.v + page * c.v_stride + at;
        const float ks = c.k_scale[page * c.k_scale_stride + kv_head], vs = value_scale(c.v_scale[page * c.v_scale_stride + kv_head]);
        float s = 0.f, v[V];
#pragma unroll
        for (int j = 0; j < V; j += 2) {
            uint32_t lo, hi;
            codes_to_half<E4M3>(*reinterpret_cast<const uint16_t *>(kp + j), lo, hi);
            const float2 k2 = unpack2<false>(lo);
            s += q[j] * k2.x + q[j + 1] * k2.y;
            codes_to_half<E4M3>(*reinterpret_cast<const uint16_t *>(vp + j), lo, hi);
            const float2 v2 = unpack2<false>(lo);
            v[j] = v2.x * vs;
            v[j + 1] = v2.y * vs;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        s *= ks;
        const float big = fmaxf(m, s), keep = m == -INFINITY ? 0.f : __expf(m - big), p = __expf(s - big);
        m = big;
        l = l * keep + p;
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] = acc[j] * keep + p * v[j];
    }
    const float inverse = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int j = 0; j < V; j += 2)
        *reinterpret_cast<uint32_t *>(a.out + id * D + lane * V + j) = pack2<BF16>(acc[j] * inverse, acc[j + 1] * inverse);
}

template <bool BF16, bool E4M3>
int launch_attention(const AttentionArgs &a, cudaStream_t s)
{
    const dim3 grid((unsigned)(((long long)a.rows.rows * a.heads + 3) / 4));
    switch (a.cache.head_dim) {
    case 64: return launch_pdl("paged_attention", attention_kernel<BF16, E4M3, 64>, grid, dim3(128), 1, 0, s, a);
    case 128: return launch_pdl("paged_attention", attention_kernel<BF16, E4M3, 128>, grid, dim3(128), 1, 0, s, a);
    default: return launch_pdl("paged_attention", attention_kernel<BF16, E4M3, 256>, grid, dim3(128), 1, 0, s, a);
    }
}

int check_sizes(const macko_kv_cache *cache, const macko_kv_rows *batch, int heads, AttentionArgs *a)
{
    if (int st = check_cache("paged_attention", cache, &a->cache)) return st;
    if (int st = check_rows("paged_attention", batch, cache->page_size, &a->rows)) return st;
    if (heads <= 0 || heads > 4096 || heads % cache->kv_heads)
        return fail(MACKO_ERR_INVALID_ARGUMENT, "paged_attention: %d heads for %d key heads", heads, cache->kv_heads);
    if (a->rows.rows > INT_MAX / heads) return fail(MACKO_ERR_SIZE_OVERFLOW, "paged_attention: %d rows of %d heads", a->rows.rows, heads);
    return MACKO_OK;
}

}  // namespace
}  // namespace macko

using namespace macko;

extern "C" {

int64_t macko_cache_attention_workspace_bytes(int64_t sequences, int64_t rows, int64_t table_width, int32_t heads, int32_t kv_heads,
                                              int32_t page_size, int32_t head_dim, int32_t one_row_each)
{
    // the refusals of macko_cache_attention, from the arguments that size it
    const macko_kv_cache cache = {reinterpret_cast<void *>(16), reinterpret_cast<void *>(16), reinterpret_cast<float *>(16), reinterpret_cast<float *>(16),
                                  INT64_MAX / 16 * 16, INT64_MAX / 16 * 16, INT64_MAX, INT64_MAX, 1, kv_heads, page_size, head_dim, MACKO_KV_INT8};
    const macko_kv_rows batch = {reinterpret_cast<const int32_t *>(16), reinterpret_cast<const int32_t *>(16),
                                 one_row_each ? nullptr : reinterpret_cast<const int32_t *>(16), table_width, table_width, sequences, rows};
    AttentionArgs a = {};
    if (check_sizes(&cache, &batch, heads, &a)) return -1;
    return 0;
}

int macko_cache_attention(const macko_kv_cache *cache, const macko_kv_rows *batch, const void *q, int64_t q_row_stride,
                          int64_t q_head_stride, int32_t type, void *out, int32_t heads, float scale, void *workspace,
                          int64_t workspace_bytes, void *stream)
{
    AttentionArgs a = {};
    if (int st = check_sizes(cache, batch, heads, &a)) return st;
    if (type != MACKO_FP16 && type != MACKO_BF16) return fail(MACKO_ERR_INVALID_ARGUMENT, "paged_attention: unknown type %d", type);
    if (a.rows.rows == 0) return MACKO_OK;
    if (!q || !out) return fail(MACKO_ERR_INVALID_ARGUMENT, "paged_attention: null pointer");
    if (!aligned(q, 16) || !aligned(out, 16) || q_row_stride % 8 || q_head_stride % 8)
        return fail(MACKO_ERR_MISALIGNED, "paged_attention: rows and heads of q and out must be 16-byte aligned");
    a.q = static_cast<const uint16_t *>(q);
    a.out = static_cast<uint16_t *>(out);
    a.q_row_stride = q_row_stride;
    a.q_head_stride = q_head_stride;
    a.heads = heads;
    a.scale = scale;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool e4m3 = cache->code == MACKO_KV_E4M3;
    if (type == MACKO_BF16) return e4m3 ? launch_attention<true, true>(a, s) : launch_attention<true, false>(a, s);
    return e4m3 ? launch_attention<false, true>(a, s) : launch_attention<false, false>(a, s);
}

}  // extern "C"
