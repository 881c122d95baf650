// What the two attention kernels over the paged cache (a few rows, many rows) and the one that joins their pieces share.
#pragma once

#include "attention_work.cuh"

namespace macko {

struct AttentionArgs {
    CacheView cache;
    RowsView rows;
    WorkShape work;
    const uint16_t *q;
    uint16_t *out;
    SplitUnit *split;        // [ctas], or null: one unit per CTA, nothing is split
    float *partial;          // [ctas][2][unit rows][head_dim + 2]
    long long q_row_stride, q_head_stride;
    int heads, unit_rows;
    float scale;             // times log2 e
    unsigned wait_limit;     // nanoseconds that a wait inside the kernel for many rows may take
};

// Rows per unit of the kernel for many rows, and its launch (no join): prompt_attention.cu.
constexpr int prompt_rows(int head_dim) { return head_dim == 256 ? 128 : 256; }
constexpr int kPromptTile = 64;
int launch_prompt_attention(const AttentionArgs &a, bool bf16, bool e4m3, cudaStream_t stream);

#ifdef __CUDACC__

__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Row ρ of a unit is row ρ / heads of its rows and head ρ % heads of its heads.
struct UnitRows {
    int first_row, queries, heads, head;   // first row of the call, rows, heads, first head
    int begin;                             // position of the first row
    __device__ __forceinline__ int rows() const { return queries * heads; }
};

__device__ __forceinline__ UnitRows unit_rows(const AttentionArgs &a, const SequenceWork &s, const Piece &p)
{
    UnitRows u;
    const WorkShape &w = a.work;
    u.first_row = s.rows.first + p.block * w.queries;
    u.queries = min(w.queries, s.rows.count - p.block * w.queries);
    u.heads = min(w.heads, w.group - p.part * w.heads);
    u.head = p.kv_head * w.group + p.part * w.heads;
    u.begin = s.rows.begin() + p.block * w.queries;
    return u;
}

// 2^-e and 2^e of a bfloat16 row's own exponent e, with which its largest value becomes 2^14 .. 2^15 in fp16; values that are not
// finite stay as they are, and e stays inside what fp32 can give back.
__device__ __forceinline__ void row_power(float most, float &down, float &up)
{
    const int e = most > 0.f && most < INFINITY ? min(max((int)(__float_as_uint(most) >> 23) - 127 - 14, -112), 113) : 0;
    down = __uint_as_float((uint32_t)(127 - e) << 23);
    up = __uint_as_float((uint32_t)(127 + e) << 23);
}

// Rows of no sequence, those before the first one's and behind the last one's, get zeros; the grid's threads share them.
__device__ __forceinline__ void clear_other_rows(const AttentionArgs &a)
{
    const RowsView &r = a.rows;
    if (r.start == nullptr) return;
    const int lo = r.sequences > 0 ? min(max(__ldcg(r.start), 0), r.rows) : r.rows;
    const int hi = r.sequences > 0 ? min(max(__ldcg(r.start + r.sequences), lo), r.rows) : r.rows;
    const long long per_row = (long long)a.heads * a.cache.head_dim / 8;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < (lo + r.rows - hi) * per_row; i += (long long)gridDim.x * blockDim.x) {
        const long long row = i / per_row, at = row < lo ? row : row - lo + hi;
        reinterpret_cast<uint4 *>(a.out)[at * per_row + i % per_row] = make_uint4(0u, 0u, 0u, 0u);
    }
}

#endif  // __CUDACC__

}  // namespace macko
