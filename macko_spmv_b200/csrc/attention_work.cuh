// How attention over the paged cache is cut into work for a fixed number of CTAs, and how the pieces are put together again.
//
// A unit is one head of the cache and the rows of one sequence that meet it together: `queries` consecutive rows of the call with `heads`
// heads each (a group of more heads than a unit holds is cut into `parts`). It walks the tokens in tiles of `tile`. Units of a sequence
// are ordered by (head, part), then by rows; block b of the rows ends at position begin + (b + 1) * queries - 1 and takes
// ceil((begin + (b + 1) * queries) / tile) tiles. All tiles of the call in this order are numbered, and in front of each unit's tiles
// `extra` numbers stand for what a unit costs whatever its length is; CTA c takes numbers [c * share, (c + 1) * share). So every CTA has
// the same work whatever the lengths are, a unit's tiles lie in consecutive CTAs, and a CTA has at most two units that are not its own
// alone: the one that began before it and the one that goes on after it. Their partial results (maximum, sum, weighted values, fp32) go
// to scratch memory, and a second small kernel puts them together.
#pragma once

#include "kv_cache.cuh"

namespace macko {

struct WorkShape {
    int queries, heads, parts;   // rows and heads of a unit, parts of a head group
    int tile;                    // tokens
    int group, kv_heads;         // heads per cache head, cache heads
    int ctas, least_share;
    int extra;                   // numbers that a unit has in front of its tiles, for the time that it takes whatever its length is
};

// Rows of a unit that goes on in the CTAs behind: what the second kernel needs. pieces 0: nothing.
struct SplitUnit {
    int first_row, rows, head, pieces;   // rows = queries * heads, packed query by query
    int heads;
    int lost;                            // 1: the CTA has given up; NaN is in all rows that it has a part in
    int unused[2];
};

// sum of floor((a * i + b) / m) for i = 0 .. n - 1; a * n + b, once a and b are below m, fits 32 bits
__host__ __device__ __noinline__ inline long long floor_sum(unsigned n, unsigned m, unsigned a, unsigned b)
{
    unsigned long long sum = 0;
    while (n > 0) {
        if (a >= m) {
            sum += (unsigned long long)(n - 1) * n / 2 * (a / m);
            a %= m;
        }
        if (b >= m) {
            sum += (unsigned long long)n * (b / m);
            b %= m;
        }
        const unsigned last = a * n + b;
        if (last < m) break;
        n = last / m;
        b = last % m;
        const unsigned t = m;
        m = a;
        a = t;
    }
    return (long long)sum;
}

// Numbers of the first `blocks` row blocks of a sequence whose rows begin at position `begin`, for one (head, part).
__host__ __device__ inline long long tiles_before(const WorkShape &w, int begin, int blocks)
{
    if (blocks == 0) return 0;
    const long long extra = (long long)w.extra * blocks;
    if (blocks == 1) return ((long long)begin + w.queries + w.tile - 1) / w.tile + extra;
    return floor_sum(blocks, w.tile, w.queries, (unsigned)begin + w.queries + w.tile - 1) + extra;
}

#ifdef __CUDACC__

// One sequence's rows in blocks.
struct SequenceWork {
    Sequence rows;
    int begin, blocks;       // begin: first position, kept inside 0 .. capacity for counting
};

__device__ __forceinline__ SequenceWork sequence_work(const WorkShape &w, const RowsView &r, const Sequence &rows)
{
    SequenceWork s;
    s.rows = rows;
    s.begin = min(max(s.rows.begin(), 0), r.capacity);
    s.blocks = (s.rows.count + w.queries - 1) / w.queries;
    return s;
}

__device__ __forceinline__ long long sequence_tiles(const WorkShape &w, const RowsView &r, const Sequence &rows)
{
    const SequenceWork s = sequence_work(w, r, rows);
    return tiles_before(w, s.begin, s.blocks) * (w.kv_heads * w.parts);
}

// A run of tiles of one unit, as one CTA walks it.
struct Piece {
    int sequence, block, kv_head, part;
    int first_tile, tiles;   // tiles [first_tile, + tiles) of the unit
    bool begins, ends;       // whether the unit begins and ends with it
    int pieces;              // CTAs that share the unit, counted where it begins
};

__device__ __forceinline__ long long quotient(long long a, long long b)   // of numbers that are not negative; most fit 32 bits
{
    return ((a | b) >> 32) == 0 ? (long long)((unsigned)a / (unsigned)b) : a / b;
}

// Walks the pieces of CTA `cta`. All lanes of a warp walk together.
struct WorkWalk {
    long long at, end, share;
    int cta, sequence, head_part, block, tile;   // where the walk is; tile: of the unit's numbers, the extra ones first
    SequenceWork s;

    __device__ void start(const WorkShape &w, const RowsView &r, int of_cta)
    {
        const int lane = threadIdx.x & 31;
        cta = of_cta;
        // the total, then the sequence with this CTA's first tile
        long long total = 0, first_own = 0;
        Sequence first_rows = {0, 0, 0};
#pragma unroll 4
        for (int i = lane; i < r.sequences; i += 32) {
            const Sequence rows = sequence_at(r, i);
            const long long own = sequence_tiles(w, r, rows);
            if (i == lane) {
                first_own = own;
                first_rows = rows;
            }
            total += own;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        share = max(quotient(total + w.ctas - 1, w.ctas), (long long)w.least_share);
        at = share * cta;
        end = min(at + share, total);
        sequence = r.sequences;
        if (at >= end) return;
        long long before = 0, base = 0;
        for (int first = 0; first < r.sequences; first += 32) {
            const long long own = first == 0 ? first_own : first + lane < r.sequences ? sequence_tiles(w, r, sequence_at(r, first + lane)) : 0;
            long long sum = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long v = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += v;
            }
            const long long lo = before + sum - own;
            const uint32_t here = __ballot_sync(0xffffffffu, at >= lo && at < lo + own);
            if (here != 0) {
                sequence = first + __ffs(here) - 1;
                base = __shfl_sync(0xffffffffu, lo, __ffs(here) - 1);
                break;
            }
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (sequence >= r.sequences) {   // the lengths have changed under the call: nothing outside the arrays is read for that
            at = end;
            return;
        }
        Sequence rows;
        if (sequence < 32) {
            rows.first = __shfl_sync(0xffffffffu, first_rows.first, sequence);
            rows.count = __shfl_sync(0xffffffffu, first_rows.count, sequence);
            rows.length = __shfl_sync(0xffffffffu, first_rows.length, sequence);
        } else {
            rows = sequence_at(r, sequence);
        }
        s = sequence_work(w, r, rows);
        const long long local = at - base, per_head = tiles_before(w, s.begin, s.blocks);
        head_part = (int)quotient(local, max(per_head, 1ll));
        const long long rest = local - head_part * per_head;
        before = 0;
        int lo = 0, hi = s.blocks;   // tiles_before(lo) <= rest < tiles_before(hi)
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            const long long t = tiles_before(w, s.begin, mid);
            if (t <= rest) {
                lo = mid;
                before = t;
            } else {
                hi = mid;
            }
        }
        block = lo;
        tile = (int)(rest - before);
    }

    // The next piece, or false. All lanes of a warp call it together, like start().
    __device__ bool next(const WorkShape &w, const RowsView &r, Piece &p)
    {
        if (at >= end) return false;
        while (s.blocks == 0 || head_part >= w.kv_heads * w.parts) {
            // the next sequence that has rows: a padded batch may have many without
            const int other = sequence + 1 + (int)(threadIdx.x & 31);
            const uint32_t with_rows = __ballot_sync(0xffffffffu, other < r.sequences && sequence_at(r, other).count > 0);
            sequence += with_rows != 0 ? __ffs(with_rows) : 32;
            if (sequence >= r.sequences) return false;
            if (with_rows == 0) continue;
            s = sequence_work(w, r, sequence_at(r, sequence));
            head_part = block = tile = 0;
        }
        const int of_unit = (int)(((long long)s.begin + (long long)(block + 1) * w.queries + w.tile - 1) / w.tile) + w.extra;
        const int taken = (int)min((long long)max(of_unit - tile, 0), end - at);
        if (tile + taken <= w.extra) {   // the unit's first tile is the next CTA's
            at = end;
            return false;
        }
        p.sequence = sequence;
        p.block = block;
        p.kv_head = head_part / w.parts;
        p.part = head_part % w.parts;
        p.first_tile = max(tile - w.extra, 0);
        p.tiles = tile + taken - w.extra - p.first_tile;
        p.begins = tile <= w.extra;
        p.ends = tile + taken >= of_unit;
        p.pieces = p.begins ? p.ends ? 1 : (int)(quotient(at + of_unit - tile - 1, share) - cta) + 1 : 0;
        at += taken;
        tile += taken;
        if (p.ends) {
            tile = 0;
            if (++block == s.blocks) {
                block = 0;
                ++head_part;
            }
        }
        return true;
    }
};

#endif  // __CUDACC__

}  // namespace macko
