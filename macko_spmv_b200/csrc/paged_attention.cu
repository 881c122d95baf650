// Attention over the paged 8-bit cache, for a few rows per sequence and head of the cache: decoding and drafted tokens.
//
//   x(t) = scale * (q . k_t) * k_scale(page) * log2 e + log2 v_scale(page)        k_t, v_t: codes
//   out  = sum 2^(x(t) - m) v_t  /  sum 2^(x(t) - m) / v_scale(page),             m = max x(t) - 15
//
// The scale of the values is part of the exponent, so the weights that meet the codes are at most 2^15 whatever the scales are. Rounding them to
// fp16 is the one rounding on the way: 2^-11 of a weight down to 2^-29 of the row's largest, 2^-40 of the largest below (with the largest at 1 it
// would be 2^-25 of it: of 30000 tokens that share a tenth of a row's weight, a hundredth was lost); sums, maxima and the accumulators are fp32. Products
// of codes with fp16 are exact in the tensor core. bfloat16 rows of q become fp16 under a power of two of their own.
//
// Bound by HBM: a code is used for 2 to 16 rows. A warp takes 16 or 32 tokens at a time from the cache straight into registers, in the
// layout that mma.m16n8k16 wants: tokens (for S^T = K Q^T) and dimensions (for O^T = V^T P^T) are its 16 rows, the call's rows its 8 columns, so that
// one step costs half of what it would the other way round. Which dimensions are "k = 2t, 2t + 1" is free as long as K and Q agree, so a
// lane loads 16 consecutive bytes of a token; bytes of two tokens are interleaved for V. The next K is asked for when this one has been
// converted, and V alike, so a warp has its 8 KB in flight all the time; the turn behind that is on its way to the L2 cache.
//
// 64 sequences of 205 to 4096 tokens, 32 heads of 128, e4m3: 229 us, 5.1 TB/s, 0.79 of what a copy moves; 131072 tokens, 8 cache heads: 61 us,
// 4.4 TB/s. 32 tokens take a warp some 550 instructions, 160 of them conversions and byte interleaving, and 168 registers leave room for 12
// warps of an SM (with 310 bytes of a thread spilled at head_dim 128; units of 16 rows, 255 registers and 8 warps: 30 to 90 at 128, 740 to 840 at 256).
// 16 warps with 16 tokens each and q in shared memory are no faster: sequences of equal length, 64 of 4096 tokens 348 against 343 us, 8192 tokens of
// one sequence 17.7 against 14.8.
#include <atomic>
#include <climits>
#include <cmath>

#include "attention_args.cuh"
#include "launch.cuh"

namespace macko {
namespace {

constexpr int kWarps = 4;
constexpr int kAhead = 1;   // turns of a warp between asking for its tokens and loading them
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kTop = 15.f;   // exponent of the largest weight: fp16 ends at 2^16

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x)
{
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// BYTES consecutive codes.
template <int BYTES> struct Codes { uint32_t w[BYTES / 4]; };

template <int BYTES>
__device__ __forceinline__ Codes<BYTES> load_codes(const uint8_t *p)
{
    Codes<BYTES> c;
    if (BYTES == 8) {
        const uint2 v = __ldcg(reinterpret_cast<const uint2 *>(p));
        c.w[0] = v.x;
        c.w[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i) {
            const uint4 v = __ldcg(reinterpret_cast<const uint4 *>(p) + i);
            c.w[4 * i] = v.x;
            c.w[4 * i + 1] = v.y;
            c.w[4 * i + 2] = v.z;
            c.w[4 * i + 3] = v.w;
        }
    }
    return c;
}

template <int BYTES>
__device__ __forceinline__ Codes<BYTES> no_codes()
{
    Codes<BYTES> c;
#pragma unroll
    for (int i = 0; i < BYTES / 4; ++i) c.w[i] = 0u;
    return c;
}

// Has `bytes` of global memory brought to the L2 cache.
__device__ __forceinline__ void prefetch(const void *p, int bytes)
{
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}

template <bool BF16, bool E4M3, int D, int RB>
__global__ void __launch_bounds__(kWarps * 32, RB == 8 && D <= 128 ? 3 : 2)
few_rows_kernel(const AttentionArgs a)
{
    constexpr int NB = RB / 8;              // blocks of 8 rows
    constexpr int MT = D == 256 ? 1 : 2;    // blocks of 16 tokens that a warp takes at a time
    constexpr int kTile = kWarps * 16 * MT;
    constexpr int KC = D / 64;              // 16-byte chunks of a key that a lane holds
    constexpr int VB = D / 8;               // bytes of a value that a lane holds
    constexpr int DT = D / 16;              // blocks of 16 dimensions
    extern __shared__ __align__(16) float merge[];   // [warps][RB][D], then maxima and sums [warps][RB]
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const RowsView &r = a.rows;
    const CacheView &c = a.cache;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int page_mask = (1 << c.page_log2) - 1;

    WorkWalk walk;
    Piece piece;
    bool more;
    if (a.split != nullptr) {
        if (tid == 0) a.split[blockIdx.x].pieces = 0;
        walk.start(a.work, r, blockIdx.x);
        more = walk.next(a.work, r, piece);
    } else {
        // one unit per CTA: sequences of one row each
        const int per_sequence = a.work.kv_heads * a.work.parts, of = blockIdx.x % per_sequence;
        walk.at = walk.end = 0;
        walk.s.rows = sequence_at(r, blockIdx.x / per_sequence);
        const int seen = min(max(walk.s.rows.length, 0), r.capacity);
        piece = Piece{(int)(blockIdx.x / per_sequence), 0, of / a.work.parts, of % a.work.parts, 0, (seen + kTile - 1) / kTile, true, true, 1};
        more = true;
    }
    while (more) {
        const UnitRows u = unit_rows(a, walk.s, piece);
        const int n_rows = u.rows();
        // table entry of the lane's block of 16 tokens, of the 32 that begin at `from`; asked for before anybody knows how many tokens
        // the sequence has
        auto entry_of = [&](int from) {
            const int token = from + (lane / MT) * kTile + (lane % MT) * 16;
            return token < r.capacity ? __ldcg(r.table + (long long)piece.sequence * r.table_stride + (token >> c.page_log2)) : -1;
        };
        const int first = piece.first_tile * kTile + warp * 16 * MT;
        const int first_entry = entry_of(first);

        // q as the B operand: row g of every block of 8, dimensions 64 c + 16 t + 4 i + 0..3 for step 4 c + i
        uint32_t q[NB][D / 16][2];
        float factor[NB][2];     // scale of rows 2t and 2t + 1
        int limit[NB][2];        // tokens that they see
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const int row = nb * 8 + g;
            const int query = row / u.heads, head = u.head + row % u.heads;
            const bool there = row < n_rows;
            const uint16_t *qp = a.q + (long long)(u.first_row + query) * a.q_row_stride + (long long)head * a.q_head_stride + 16 * t;
#pragma unroll
            for (int ch = 0; ch < KC; ++ch) {
                uint4 lo = make_uint4(0u, 0u, 0u, 0u), hi = lo;
                if (there) {
                    lo = __ldcg(reinterpret_cast<const uint4 *>(qp + 64 * ch));
                    hi = __ldcg(reinterpret_cast<const uint4 *>(qp + 64 * ch) + 1);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    q[nb][4 * ch + j / 2][j & 1] = (&lo.x)[j];
                    q[nb][4 * ch + 2 + j / 2][j & 1] = (&hi.x)[j];
                }
            }
            float own = 1.f;
            if (BF16) {
                float most = 0.f;
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    const float2 f = unpack2<true>((&q[nb][0][0])[i]);
                    most = fmaxf(most, fmaxf(fabsf(f.x), fabsf(f.y)));
                }
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                float down;
                row_power(most, down, own);
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    const float2 f = unpack2<true>((&q[nb][0][0])[i]);
                    (&q[nb][0][0])[i] = pack2<false>(f.x * down, f.y * down);
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                factor[nb][i] = __shfl_sync(0xffffffffu, own, 4 * (2 * t + i)) * a.scale;
                const int other = nb * 8 + 2 * t + i;
                limit[nb][i] = other < n_rows ? min(u.begin + other / u.heads + 1, r.capacity) : 0;
            }
        }
        const int all_see = min(u.begin + 1, r.capacity);                       // tokens before this are seen by every row
        const int end = max(0, min(u.begin + u.queries, r.capacity));           // and none from here on by any

        float m[NB][2], l[NB][2], o[DT][NB][4];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            m[nb][0] = m[nb][1] = -INFINITY;
            l[nb][0] = l[nb][1] = 0.f;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d][nb][0] = o[d][nb][1] = o[d][nb][2] = o[d][nb][3] = 0.f;
        }

        const int stop = min(end, (piece.first_tile + piece.tiles) * kTile);
        const long long head_at = ((long long)piece.kv_head << c.page_log2) * D;
        // Of the warp's next 32 blocks of 16 tokens, one per lane: where their codes begin, in units of 16 bytes, and what the softmax
        // needs of their page's scales.
        bool there_of_lane = false;
        uint32_t k_of_lane = 0u, v_of_lane = 0u;
        float ks_of_lane = 0.f, shift_of_lane = 0.f, inverse_of_lane = 0.f;
        Codes<16> kc[MT][2][KC];
        Codes<VB> vc[MT][4];
        auto fetch_pages = [&](int from, int page) {
            const int token = from + (lane / MT) * kTile + (lane % MT) * 16;
            there_of_lane = token < end && (unsigned)page < (unsigned)c.pages;
            if (there_of_lane) {
                const long long off = head_at + (long long)(token & page_mask) * D;
                k_of_lane = (uint32_t)((page * c.k_stride + off) >> 4);
                v_of_lane = (uint32_t)((page * c.v_stride + off) >> 4);
                const float vs = value_scale(__ldcg(c.v_scale + page * c.v_scale_stride + piece.kv_head));
                ks_of_lane = __ldcg(c.k_scale + page * c.k_scale_stride + piece.kv_head);
                shift_of_lane = __log2f(vs);
                inverse_of_lane = inverse_scale(vs);
            }
        };
        const uint8_t *const k_base = c.k + 16 * t + g * D, *const v_base = c.v + VB * g + 2 * t * D;
        // `whole`: all of the warp's tokens are there
        auto load_k = [&](int token, int index, int mt, bool whole) {
            const int from = index * MT + mt;
            const uint8_t *base = k_base + 16ull * __shfl_sync(0xffffffffu, k_of_lane, from);
            const bool there = whole || __shfl_sync(0xffffffffu, (int)there_of_lane, from);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int ch = 0; ch < KC; ++ch) {
                    if (whole || (there && token + mt * 16 + g + 8 * h < end)) kc[mt][h][ch] = load_codes<16>(base + 8 * h * D + 64 * ch);
                    else kc[mt][h][ch] = no_codes<16>();
                }
        };
        auto load_v = [&](int token, int index, int mt, bool whole) {
            const int from = index * MT + mt;
            const uint8_t *base = v_base + 16ull * __shfl_sync(0xffffffffu, v_of_lane, from);
            const bool there = whole || __shfl_sync(0xffffffffu, (int)there_of_lane, from);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = (i & 1) + 8 * (i >> 1);
                if (whole || (there && token + mt * 16 + 2 * t + row < end)) vc[mt][i] = load_codes<VB>(base + row * D);
                else vc[mt][i] = no_codes<VB>();
            }
        };
        auto is_whole = [&](int token, int index) {
            return __all_sync(0xffffffffu, there_of_lane || lane / MT != index) && token + 16 * MT <= end;
        };
        // the tokens of one of the warp's turns behind, K and V, to the L2 cache: the registers hold no more than one turn, and a load
        // from memory takes longer than a turn
        auto ask = [&](int index) {
            if (lane / MT == index && there_of_lane) {
                prefetch(c.k + 16ull * k_of_lane, 16 * D);
                prefetch(c.v + 16ull * v_of_lane, 16 * D);
            }
        };
        constexpr int kPerFetch = 32 / MT;
        int index = 0;
        bool whole = false;   // the current turn's tokens are all there
        if (first < stop) {
            fetch_pages(first, first_entry);
            whole = is_whole(first, 0);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) load_k(first, 0, mt, whole);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) load_v(first, 0, mt, whole);
#pragma unroll
            for (int i = 1; i <= kAhead; ++i) ask(i);
        }
        for (int token = first; token < stop; token += kTile) {
            float x[MT][NB][4], inverse[MT];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) x[mt][nb][0] = x[mt][nb][1] = x[mt][nb][2] = x[mt][nb][3] = 0.f;
#pragma unroll
                for (int ch = 0; ch < KC; ++ch)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t a0, a1, a2, a3;
                        codes_to_half<E4M3>(kc[mt][0][ch].w[i], a0, a2);
                        codes_to_half<E4M3>(kc[mt][1][ch].w[i], a1, a3);
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) mma(x[mt][nb], a0, a1, a2, a3, q[nb][4 * ch + i][0], q[nb][4 * ch + i][1]);
                    }
            }
            // what the softmax needs of this slice's pages, before the next ones may take their place
            float k_scale[MT], shift[MT];
            bool there[MT];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                const int from = index * MT + mt;
                k_scale[mt] = __shfl_sync(0xffffffffu, ks_of_lane, from);
                shift[mt] = __shfl_sync(0xffffffffu, shift_of_lane, from);
                inverse[mt] = __shfl_sync(0xffffffffu, inverse_of_lane, from);
                there[mt] = whole || __shfl_sync(0xffffffffu, (int)there_of_lane, from);
            }
            const int next = token + kTile;
            const bool go_on = next < stop;
            if (++index == kPerFetch && go_on) {
                index = 0;
                fetch_pages(next, entry_of(next));
            }
            bool next_whole = false;
            if (go_on) {
                next_whole = is_whole(next, index);
                if (next_whole) {
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) load_k(next, index, mt, true);
                } else {
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) load_k(next, index, mt, false);
                }
                ask(index + kAhead);
            }

            float top[NB][2];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) top[nb][0] = top[nb][1] = -INFINITY;
            const bool all_seen = token + 16 * MT <= all_see;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float &v = x[mt][nb][i];
                        v = v * (k_scale[mt] * factor[nb][i & 1]) + shift[mt];
                        if (!there[mt] || (!all_seen && token + mt * 16 + g + 8 * (i >> 1) >= limit[nb][i & 1])) v = -INFINITY;
                        top[nb][i & 1] = fmaxf(top[nb][i & 1], v);
                    }
            }
            bool grown = false;
            float keep[NB][2], base[NB][2];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float &v = top[nb][i];
#pragma unroll
                    for (int s = 4; s < 32; s <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, s));
                    v = fmaxf(__fadd_ru(v, -kTop), m[nb][i]);   // up: a weight is at most 2^15 also where fp32 has no such difference
                    base[nb][i] = v == -INFINITY ? 0.f : v;
                    keep[nb][i] = exp2_fast(m[nb][i] - base[nb][i]);
                    grown |= v != m[nb][i];
                    m[nb][i] = v;
                }
            if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    l[nb][0] *= keep[nb][0];
                    l[nb][1] *= keep[nb][1];
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[d][nb][i] *= keep[nb][i & 1];
                }
            }
            uint32_t p[MT][NB][2];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[mt][nb][i] = exp2_fast(x[mt][nb][i] - base[nb][i & 1]);
                    // tokens that a row does not see may have any scale: they add nothing
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float sum = x[mt][nb][i] + x[mt][nb][2 + i];
                        l[nb][i] += sum == 0.f ? 0.f : sum * inverse[mt];
                    }
                    p[mt][nb][0] = transpose8x8(pack2<false>(x[mt][nb][0], x[mt][nb][1]));
                    p[mt][nb][1] = transpose8x8(pack2<false>(x[mt][nb][2], x[mt][nb][3]));
                }
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int w = 0; w < VB / 4; ++w) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const uint32_t select = half ? 0x7362u : 0x5140u;
                        uint32_t a0, a1, a2, a3;
                        codes_to_half<E4M3>(__byte_perm(vc[mt][0].w[w], vc[mt][1].w[w], select), a0, a1);
                        codes_to_half<E4M3>(__byte_perm(vc[mt][2].w[w], vc[mt][3].w[w], select), a2, a3);
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) mma(o[2 * w + half][nb], a0, a1, a2, a3, p[mt][nb][0], p[mt][nb][1]);
                    }
                }
            if (next_whole) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) load_v(next, index, mt, true);
            } else if (go_on) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) load_v(next, index, mt, false);
            }
            whole = next_whole;
        }

        // the warps' results together: rows 2t, 2t + 1 of every block, dimensions g * D / 8 + 2 d + (0, 1)
        float *maxima = merge + kWarps * RB * D, *sums = maxima + kWarps * RB;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float v = l[nb][i];
#pragma unroll
                for (int s = 4; s < 32; s <<= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
                const int row = nb * 8 + 2 * t + i;
                if (g == 0) {
                    maxima[warp * RB + row] = m[nb][i];
                    sums[warp * RB + row] = v;
                }
                float2 *to = reinterpret_cast<float2 *>(merge + (warp * RB + row) * D + g * VB);
#pragma unroll
                for (int d = 0; d < DT; ++d) to[d] = make_float2(o[d][nb][i], o[d][nb][2 + i]);
            }
        __syncthreads();
        const bool alone = piece.begins && piece.ends;
        float *partial = alone ? nullptr : a.partial + ((long long)blockIdx.x * 2 + (piece.begins ? 1 : 0)) * RB * (D + 2);
        for (int i = tid; i < n_rows * (D / 4); i += kWarps * 32) {
            const int row = i / (D / 4), d = 4 * (i % (D / 4));
            float most = -INFINITY, sum = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) most = fmaxf(most, maxima[w * RB + row]);
            const float base = most == -INFINITY ? 0.f : most;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float f = exp2_fast(maxima[w * RB + row] - base);
                const float4 x = *reinterpret_cast<const float4 *>(merge + (w * RB + row) * D + d);
                sum += f * sums[w * RB + row];
                v.x += f * x.x;
                v.y += f * x.y;
                v.z += f * x.z;
                v.w += f * x.w;
            }
            if (alone) {
                const float inverse = sum == 0.f ? 0.f : 1.f / sum;
                const uint2 packed = make_uint2(pack2<BF16>(v.x * inverse, v.y * inverse), pack2<BF16>(v.z * inverse, v.w * inverse));
                const long long to = ((long long)(u.first_row + row / u.heads) * a.heads + u.head + row % u.heads) * D + d;
                *reinterpret_cast<uint2 *>(a.out + to) = packed;
            } else {
                *reinterpret_cast<float4 *>(partial + row * D + d) = v;
                if (d == 0) {
                    partial[RB * D + row] = most;
                    partial[RB * D + RB + row] = sum;
                }
            }
        }
        if (!alone && piece.begins && tid == 0)
            a.split[blockIdx.x] = SplitUnit{u.first_row, n_rows, u.head, piece.pieces, u.heads, 0, {0, 0}};
        __syncthreads();
        more = walk.next(a.work, r, piece);
    }

    clear_other_rows(a);
}

// Units that lie in several CTAs. Every block makes the list of them (the CTAs with whose share they begin); their rows are dealt out, to
// warps where there are many, else to blocks, whose warps share a row's pieces.
constexpr int kMostCtas = 1024;

template <bool BF16, int D>
__global__ void __launch_bounds__(256)
join_kernel(const AttentionArgs a)
{
    constexpr int V = D / 32;   // dimensions of a lane: 2, 4 or 8
    __shared__ float parts[8][D + 2];
    __shared__ int list[kMostCtas], counts[9];
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, ctas = a.work.ctas;
    // in order, so that every block has the same list: each warp a range of CTAs
    const int range = (ctas + 255) / 256;
    uint32_t split = 0u;   // of this thread's CTAs
    for (int i = 0; i < range; ++i) {
        const int cta = (warp * 32 + lane) * range + i;
        if (cta < ctas && __ldcg(&a.split[cta].pieces) > 0) split |= 1u << i;
    }
    int own = __popc(split), sum = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
    }
    if (lane == 31) counts[warp] = sum;
    __syncthreads();
    int at = sum - own, units = 0;
    for (int w = 0; w < 8; ++w) {
        if (w < warp) at += counts[w];
        units += counts[w];
    }
    for (int i = 0; i < range; ++i)
        if (split >> i & 1u) list[at++] = (warp * 32 + lane) * range + i;
    __syncthreads();
    const int rows = units * a.unit_rows, stride = a.unit_rows * (D + 2);
    const bool shared = rows <= (int)gridDim.x * 2;   // a row for a block, not for a warp
    for (int item = shared ? (int)blockIdx.x : (int)blockIdx.x * 8 + warp; item < rows; item += shared ? gridDim.x : gridDim.x * 8) {
        const int cta = list[item / a.unit_rows], row = item % a.unit_rows;
        const int4 s = __ldcg(reinterpret_cast<const int4 *>(a.split + cta));   // first row, rows, head, pieces
        if (row >= s.y) continue;
        const int unit_heads = __ldcg(&a.split[cta].heads);
        const int member = shared ? warp : 0, members = shared ? 8 : 1, pieces = s.w;
        float m = -INFINITY, l = 0.f, o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = 0.f;
        constexpr int U = 4;
        for (int p0 = member; p0 < pieces; p0 += U * members) {
            float pm[U], pl[U], po[U][V];
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int p = p0 + i * members;
                pm[i] = -INFINITY;
                pl[i] = 0.f;
#pragma unroll
                for (int j = 0; j < V; ++j) po[i][j] = 0.f;
                if (p < pieces) {
                    // the first piece is the second result of its CTA, the others are the first of theirs
                    const float *from = a.partial + ((long long)(cta + p) * 2 + (p == 0)) * stride;
                    pm[i] = __ldcg(from + a.unit_rows * D + row);
                    pl[i] = __ldcg(from + a.unit_rows * D + a.unit_rows + row);
#pragma unroll
                    for (int j = 0; j < V; j += 2) {
                        const float2 x = __ldcg(reinterpret_cast<const float2 *>(from + row * D + lane * V + j));
                        po[i][j] = x.x;
                        po[i][j + 1] = x.y;
                    }
                }
            }
            float most = m;
#pragma unroll
            for (int i = 0; i < U; ++i) most = fmaxf(most, pm[i]);
            const float base = most == -INFINITY ? 0.f : most, keep = exp2_fast(m - base);
            m = most;
            l *= keep;
#pragma unroll
            for (int j = 0; j < V; ++j) o[j] *= keep;
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const float f = exp2_fast(pm[i] - base);
                l += f * pl[i];
#pragma unroll
                for (int j = 0; j < V; ++j) o[j] += f * po[i][j];
            }
        }
        if (shared) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < V; ++j) parts[warp][lane * V + j] = o[j];
            if (lane == 0) {
                parts[warp][D] = m;
                parts[warp][D + 1] = l;
            }
            __syncthreads();
            if (warp != 0) continue;
            float most = m;
            for (int w = 1; w < 8; ++w) most = fmaxf(most, parts[w][D]);
            const float base = most == -INFINITY ? 0.f : most, keep = exp2_fast(m - base);
            l *= keep;
#pragma unroll
            for (int j = 0; j < V; ++j) o[j] *= keep;
            for (int w = 1; w < 8; ++w) {
                const float f = exp2_fast(parts[w][D] - base);
                l += f * parts[w][D + 1];
#pragma unroll
                for (int j = 0; j < V; ++j) o[j] += f * parts[w][lane * V + j];
            }
        }
        const float inverse = l == 0.f ? 0.f : 1.f / l;
        uint16_t *to = a.out + ((long long)(s.x + row / unit_heads) * a.heads + s.z + row % unit_heads) * D + lane * V;
#pragma unroll
        for (int j = 0; j < V; j += 2) *reinterpret_cast<uint32_t *>(to + j) = pack2<BF16>(o[j] * inverse, o[j + 1] * inverse);
    }
}

// The same for units of many rows, which lie in two or three CTAs: a warp has four rows at a time.
template <bool BF16, int D>
__global__ void __launch_bounds__(512)
join_many_kernel(const AttentionArgs a)
{
    constexpr int V = D / 32, R = 4;
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int4 *at = reinterpret_cast<const int4 *>(a.split + blockIdx.x);
    const int4 s = __ldcg(at);   // first row, rows, head, pieces
    const int2 more = __ldcg(reinterpret_cast<const int2 *>(at + 1));   // heads, lost
    const int unit_heads = more.x, lane = threadIdx.x & 31;
    const int row0 = (blockIdx.y * 16 + (threadIdx.x >> 5)) * R;
    if (s.w == 0 || row0 >= s.y || more.y != 0) return;   // lost: NaN is there already
    const int stride = a.unit_rows * (D + 2);
    float m[R], l[R], o[R][V];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) o[i][j] = 0.f;
    }
    int lost = 0;
    for (int p = 0; p < s.w; ++p) {
        // the first piece is the second result of its CTA, the others are the first of theirs; rows behind the unit's have whatever
        // was there: they are not written
        const float *from = a.partial + ((long long)(blockIdx.x + p) * 2 + (p == 0)) * stride;
        lost |= __ldcg(&a.split[blockIdx.x + p].lost);
        float pm[R], pl[R], po[R][V];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            pm[i] = __ldcg(from + a.unit_rows * D + row0 + i);
            pl[i] = __ldcg(from + a.unit_rows * D + a.unit_rows + row0 + i);
#pragma unroll
            for (int j = 0; j < V; j += 2) {
                const float2 x = __ldcg(reinterpret_cast<const float2 *>(from + (row0 + i) * D + lane * V + j));
                po[i][j] = x.x;
                po[i][j + 1] = x.y;
            }
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const float most = fmaxf(m[i], pm[i]), base = most == -INFINITY ? 0.f : most;
            const float keep = exp2_fast(m[i] - base), f = exp2_fast(pm[i] - base);
            m[i] = most;
            l[i] = l[i] * keep + f * pl[i];
#pragma unroll
            for (int j = 0; j < V; ++j) o[i][j] = o[i][j] * keep + f * po[i][j];
        }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int row = row0 + i;
        if (row >= s.y) break;
        const float inverse = lost != 0 ? __uint_as_float(0x7fffffffu) : l[i] == 0.f ? 0.f : 1.f / l[i];
        uint16_t *to = a.out + ((long long)(s.x + row / unit_heads) * a.heads + s.z + row % unit_heads) * D + lane * V;
#pragma unroll
        for (int j = 0; j < V; j += 2) *reinterpret_cast<uint32_t *>(to + j) = pack2<BF16>(o[i][j] * inverse, o[i][j + 1] * inverse);
    }
}

std::atomic<unsigned> g_wait_limit{2000000000u};   // nanoseconds

int check_sizes(const macko_kv_cache *cache, const macko_kv_rows *batch, int heads, AttentionArgs *a)
{
    if (int st = check_cache("paged_attention", cache, &a->cache)) return st;
    if (int st = check_rows("paged_attention", batch, cache->page_size, &a->rows)) return st;
    if (heads <= 0 || heads > 4096 || heads % cache->kv_heads)
        return fail(MACKO_ERR_INVALID_ARGUMENT, "paged_attention: %d heads for %d key heads", heads, cache->kv_heads);
    if (a->rows.rows > INT_MAX / heads) return fail(MACKO_ERR_SIZE_OVERFLOW, "paged_attention: %d rows of %d heads", a->rows.rows, heads);
    return MACKO_OK;
}

// Which launch runs, and what it keeps in the workspace: host arithmetic on sizes alone.
struct Launch {
    WorkShape work;
    int unit_rows;      // 8 or 16; 128 or more: the kernel for many rows
    int ctas, smem, sm_count;
    bool split;
    int64_t split_bytes, partial_bytes;
};

int plan_launch(const AttentionArgs &a, int heads, int sm_count, Launch *l)
{
    const int group = heads / a.cache.kv_heads, d = a.cache.head_dim;
    const bool one_each = a.rows.start == nullptr;
    // rows that a head of the cache meets in a sequence, as far as the host knows: on average
    const int64_t mean = one_each ? group : ((int64_t)a.rows.rows * group + a.rows.sequences - 1) / (a.rows.sequences > 0 ? a.rows.sequences : 1);
    // The kernel for many rows takes 128 or 256 as long as one; the other reads and converts the cache once for 16. 16 sequences of 8000
    // tokens, head_dim 128, 12 / 32 / 40 / 64 rows: 69 / 128 / 180 / 235 us against 134 / 141 / 142 / 142; 4 of 2000, 32 rows: 21 / 26; head_dim 64,
    // 32 / 40 / 64 rows: 92 / 131 / 170 against 122 / 123 / 124; head_dim 256, 16 / 24 / 32 rows: 158 / 286 / 290 against 202 / 206 / 208, and 24 rows of
    // 1 of 8000, 4 of 2000, 16 of 1000: 36 / 38 / 65 against 65 / 39 / 50. (So at 256 a few sequences would have a higher limit, many a lower one.)
    // The mean takes in sequences without rows and single tokens, and one kernel serves the call: 8 heads of 128, a prompt of 4096 tokens with 300 sequences
    // without rows 261 us, bare 90; with 200 single tokens over 4000 each 621 together, 269 and 91 in two calls; with 60 of them 367, 93 and 90.
    const bool prompt = !one_each && mean > (d == 256 ? 24 : 32);
    // Units of 8 rows where they suffice: 16 sequences of 8000 tokens, 8 rows 58 us against 68 with units of 16, 10 rows 97 against 69.
    const int rows = prompt ? prompt_rows(d) : mean <= 8 ? 8 : 16;
    l->unit_rows = rows;
    l->work.heads = group < rows ? group : rows;
    l->work.parts = (group + l->work.heads - 1) / l->work.heads;
    l->work.queries = one_each ? 1 : rows / l->work.heads;
    l->work.tile = prompt ? kPromptTile : kWarps * 16 * (d == 256 ? 1 : 2);
    l->work.group = group;
    l->work.kv_heads = a.cache.kv_heads;
    // A CTA has at least so many numbers. One sequence of 32 heads: 1056 tokens 12.1 us with one (128 tokens), 13.6 with two, 16.7 with four; many
    // rows: 512 of a prompt 25.4 with four (of 64 tokens) or two, 27.6 with eight, 8 pieces of 100 rows 17.9 / 18.2 / 23.6.
    l->work.least_share = prompt ? 4 : 1;
    // What a unit costs by itself (its rows, the first loads, its epilogue) is that of some 256 tokens more. With 0 / 128 / 256 / 384 tokens,
    // us: 64 sequences of 205 to 4096 tokens, 32 heads of 128, 273 / 223 / 201 / 202; of 8 heads of 64 up to 2048 tokens 45 / 32 / 29 / 29;
    // of 8 heads of 256, 256 tokens 113, 384 109. Many rows, 0 / 128 / 256 / 512: a prompt of 4096, 237 / 222 / 213 / 215; 32 pieces of up to 40
    // rows 69 / 51 / 50 / 54.
    l->work.extra = 256 / l->work.tile;
    l->smem = (kWarps * rows * d + 2 * kWarps * rows) * 4;
    l->sm_count = sm_count < kMostCtas / 3 ? sm_count : kMostCtas / 3;
    const int64_t units = (int64_t)a.rows.sequences * a.cache.kv_heads * l->work.parts;
    // One CTA per unit where the table has room for few tokens: shares and the second kernel take some microseconds. Tables of 200 / 512 /
    // 1024 / 2048 tokens, one sequence of 32 heads: 6.0 / 8.7 / 14.2 / 25.1 us against 11.4 / 11.6 / 12.1 / 14.4; 16 sequences of 8 cache
    // heads, 512 / 1024: 10.7 / 17.2 against 14.2 / 16.5; 64 such: 16.0 / 25.3 against 21.9 / 27.0. (The two meet between 512 and 1024: at the limit itself
    // shares are the faster ones of the first two.)
    l->split = !(one_each && a.rows.capacity <= 1024);
    l->ctas = l->split ? l->sm_count * (prompt ? 1 : rows == 8 && d <= 128 ? 3 : 2) : 0;
    if (!l->split) {
        if (units > INT_MAX) return fail(MACKO_ERR_SIZE_OVERFLOW, "paged_attention: too many sequences and heads");
        l->ctas = (int)units;
    }
    l->work.ctas = l->ctas;
    l->split_bytes = l->split ? (int64_t)l->ctas * sizeof(SplitUnit) : 0;
    l->partial_bytes = l->split ? (int64_t)l->ctas * 2 * rows * (d + 2) * 4 : 0;
    return MACKO_OK;
}

template <bool BF16, bool E4M3, int D, int RB>
int launch_few(const AttentionArgs &a, const Launch &l, cudaStream_t s)
{
    static bool raised[kMaxDevices];   // dynamic shared memory above 48 KB is allowed per kernel and device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && l.smem > 40 * 1024 && (dev >= kMaxDevices || !raised[dev])) {
        e = cudaFuncSetAttribute(few_rows_kernel<BF16, E4M3, D, RB>, cudaFuncAttributeMaxDynamicSharedMemorySize, l.smem);
        if (e == cudaSuccess && dev < kMaxDevices) raised[dev] = true;
    }
    if (e != cudaSuccess) return fail(MACKO_ERR_CUDA, "paged_attention: %s", cudaGetErrorString(e));
    if (int st = launch_pdl("paged_attention", few_rows_kernel<BF16, E4M3, D, RB>, dim3(l.ctas), dim3(kWarps * 32), 1, l.smem, s, a)) return st;
    if (!l.split) return MACKO_OK;
    return launch_pdl("paged_attention", join_kernel<BF16, D>, dim3(2 * l.sm_count), dim3(256), 1, 0, s, a);
}

template <bool BF16, bool E4M3, int D>
int launch_rows(const AttentionArgs &a, const Launch &l, cudaStream_t s)
{
    if (l.unit_rows >= 128) {
        if (int st = launch_prompt_attention(a, BF16, E4M3, s)) return st;
        return launch_pdl("paged_attention", join_many_kernel<BF16, D>, dim3(l.ctas, l.unit_rows / 64), dim3(512), 1, 0, s, a);
    }
    return l.unit_rows == 8 ? launch_few<BF16, E4M3, D, 8>(a, l, s) : launch_few<BF16, E4M3, D, 16>(a, l, s);
}

template <bool BF16, bool E4M3>
int launch_attention(const AttentionArgs &a, const Launch &l, cudaStream_t s)
{
    switch (a.cache.head_dim) {
    case 64: return launch_rows<BF16, E4M3, 64>(a, l, s);
    case 128: return launch_rows<BF16, E4M3, 128>(a, l, s);
    default: return launch_rows<BF16, E4M3, 256>(a, l, s);
    }
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
                                  1ll << 36, 1ll << 36, 1ll << 40, 1ll << 40, 1, kv_heads, page_size, head_dim, MACKO_KV_INT8};
    const macko_kv_rows batch = {reinterpret_cast<const int32_t *>(16), reinterpret_cast<const int32_t *>(16),
                                 one_row_each ? nullptr : reinterpret_cast<const int32_t *>(16), table_width, table_width, sequences, rows};
    AttentionArgs a = {};
    const DeviceInfo *dev = nullptr;
    Launch l;
    if (check_sizes(&cache, &batch, heads, &a)) return -1;
    if (rows == 0) return 0;
    if (current_device_info(&dev) || plan_launch(a, heads, dev->sm_count, &l)) return -1;
    return l.split_bytes + l.partial_bytes;
}

int macko_cache_attention(const macko_kv_cache *cache, const macko_kv_rows *batch, const void *q, int64_t q_row_stride,
                          int64_t q_head_stride, int32_t type, void *out, int32_t heads, float scale, void *workspace,
                          int64_t workspace_bytes, void *stream)
{
    AttentionArgs a = {};
    if (int st = check_sizes(cache, batch, heads, &a)) return st;
    if (type != MACKO_FP16 && type != MACKO_BF16) return fail(MACKO_ERR_INVALID_ARGUMENT, "paged_attention: unknown type %d", type);
    if (!std::isfinite(scale * kLog2e)) return fail(MACKO_ERR_INVALID_ARGUMENT, "paged_attention: scale %g", (double)scale);
    if (a.rows.rows == 0) return MACKO_OK;
    if (!q || !out) return fail(MACKO_ERR_INVALID_ARGUMENT, "paged_attention: null pointer");
    if (!aligned(q, 16) || !aligned(out, 16) || !aligned(workspace, 16) || q_row_stride % 8 || q_head_stride % 8)
        return fail(MACKO_ERR_MISALIGNED, "paged_attention: rows and heads of q, out and the workspace must be 16-byte aligned");
    const DeviceInfo *dev = nullptr;
    if (int st = current_device_info(&dev)) return st;
    Launch l;
    if (int st = plan_launch(a, heads, dev->sm_count, &l)) return st;
    if (workspace_bytes < l.split_bytes + l.partial_bytes || (!workspace && l.split))
        return fail(MACKO_ERR_WORKSPACE, "paged_attention: %lld bytes of workspace, %lld needed", (long long)workspace_bytes,
                    (long long)(l.split_bytes + l.partial_bytes));
    a.work = l.work;
    a.q = static_cast<const uint16_t *>(q);
    a.out = static_cast<uint16_t *>(out);
    a.split = l.split ? static_cast<SplitUnit *>(workspace) : nullptr;
    a.partial = l.split ? reinterpret_cast<float *>(static_cast<char *>(workspace) + l.split_bytes) : nullptr;
    a.q_row_stride = q_row_stride;
    a.q_head_stride = q_head_stride;
    a.heads = heads;
    a.unit_rows = l.unit_rows;
    a.scale = scale * kLog2e;
    a.wait_limit = g_wait_limit.load(std::memory_order_relaxed);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool e4m3 = cache->code == MACKO_KV_E4M3;
    if (type == MACKO_BF16) return e4m3 ? launch_attention<true, true>(a, l, s) : launch_attention<true, false>(a, l, s);
    return e4m3 ? launch_attention<false, true>(a, l, s) : launch_attention<false, false>(a, l, s);
}

int macko_cache_attention_wait_limit(int64_t nanoseconds)
{
    if (nanoseconds < 0 || nanoseconds > 2000000000)
        return fail(MACKO_ERR_INVALID_ARGUMENT, "paged_attention: a limit of %lld nanoseconds (0 .. 2000000000)", (long long)nanoseconds);
    g_wait_limit.store((unsigned)nanoseconds, std::memory_order_relaxed);
    return MACKO_OK;
}

}  // extern "C"
