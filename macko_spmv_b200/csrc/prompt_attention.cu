// Attention over the paged 8-bit cache, for many rows per sequence and head of the cache: prompts and pieces of prompts.
//
//   x(t) = scale * (q . k_t) * k_scale(page) * log2 e + log2 v_scale(page)        k_t, v_t: codes
//   out  = sum 2^(x(t) - m) v_t  /  sum 2^(x(t) - m) / v_scale(page)
//
// as in the kernel for a few rows. One CTA per SM walks its share of the call's tiles (attention_work.cuh): units of 256 packed rows (rows
// of the call times heads of a group) in two halves of 128, tiles of 64 tokens. Five groups of warps:
//
//   0, 1   softmax of one half each, one row per thread: S from tensor memory, maximum, 2^x, P as fp16 over S in tensor memory; the
//          accumulator is rescaled there when the maximum has grown by more than kLag, so that a row's largest weight is 2^7 to 2^15: fp16 rounds
//          weights by 2^-11 of themselves down to 2^-21 of the largest, by 2^-32 of the largest below
//   2, 3   keys and values: codes from shared memory to fp16 (exact) in shared memory, in the 128-byte swizzle, three stages each
//   4      one warp for each half that issues its tcgen05.mma: S = Q K^T from shared memory, O += P V with P from tensor memory and V as it
//          lies (token by token: its "N" dimension is the contiguous one); two that fetch the codes of 16 tokens at a time with bulk
//          copies, one of them with the scales of their pages and after finding the CTA's next piece
//
// Tensor memory holds two S of 64 columns and one O for each half, 512 columns at head_dim 128: S of the tile behind is there before
// the softmax of this one is done. (With one S of 128 columns a half waited for its P to go through the tensor core and for the next S,
// 1900 of 5400 cycles for 128 tokens.)
//
// 4 pieces of up to 512 rows over up to 16384 tokens, 32/8 heads of 128, int8: 339 us, 790 TFLOP/s (0.47 of a cuBLAS product in a burst);
// a 4096-token prompt, 32 heads, e4m3: 213 us, 644 TFLOP/s. The tensor pipe is active 42 % of the time, a scheduler issues 0.56 instructions
// a cycle, 1360 for a tile. What bounds it is the chain from S through a half's softmax and P to the next S: with neither softmax
// arithmetic nor conversions the first case took 279 of 333 us, without the products as well 182 (a wait for what is there already takes
// 100 to 150 cycles). Tried without gain: 2^x of a part of the scores on the FMA pipe, other lengths of sleep while waiting.
//
// The warps that fetch codes look at the clock when they wait, one of them until all others have left. Where one waits too long, no wait of the CTA
// goes on: no copy is started any more, and the working warps leave their piece and then their loop, each as a whole, after a tile at most of whatever
// is there (all addresses come from the piece); tensor memory is given back behind what was issued. The rows that the CTA has a part in are filled with
// NaN, and the kernel that joins pieces leaves them so.
#include "attention_args.cuh"
#include "launch.cuh"

namespace macko {
namespace {

constexpr int kThreads = 640;
constexpr int kTile = kPromptTile;
constexpr int kGroups = kTile / 16;     // blocks of 16 tokens: each lies on one page
constexpr int kConstSlots = 16;         // scales are fetched at most 9 tiles ahead of the softmax (codes, K, S)
constexpr float kLeastFactor = 1e-36f;  // a score times nothing is still minus infinity where it is masked
constexpr float kTop = 15.f, kLag = 8.f;  // exponents of the largest weight, which fp16 ends behind, and of what a maximum may lag
                                          // (by 4: pieces 340 instead of 333 us)
constexpr float kFar = 1048576.f;       // 2^20, where steps of fp32 are an eighth
constexpr uint32_t kSleep = 20000u;     // nanoseconds that a warp sleeps at a time while it waits
constexpr int kWorkers = 19;            // warps that are given the CTA's pieces by the one that finds them

// Shared memory, from a 1024-byte boundary: Q of the halves, K and V stages, each as [64 dimensions][rows][128 bytes]; codes of K and V.
// At head_dim 256 O takes 256 columns of tensor memory: units have one half, and there is room for two stages and for one of codes.
template <int D> struct Layout {
    static constexpr int kHalves = D == 256 ? 1 : 2, kRows = 128 * kHalves;
    static constexpr int kStages = D == 256 ? 2 : 3, kCodeStages = D == 256 ? 1 : 3;
    static constexpr int kHalf = 128 * D * 2, kStage = kTile * D * 2, kCodes = kTile * D;
    static constexpr int kQ = 0, kK = kHalves * kHalf, kV = kK + kStages * kStage, kKCodes = kV + kStages * kStage, kVCodes = kKCodes + kCodeStages * kCodes;
    static constexpr int kBytes = kVCodes + kCodeStages * kCodes + 1024;
};

// A place in a ring of N and how often it has been around, modulo 2.
template <int N> struct Ring {
    int stage = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void next()
    {
        if (++stage == N) {
            stage = 0;
            phase ^= 1u;
        }
    }
};

// Barriers with several in a row: of a half, of a stage, of half * 2 + S buffer, of a slot. A wait tells a phase from its neighbours
// only: whoever waits for one knows that the one before has come and that the one behind it needs the waiter. (So O += P V has two
// barriers for each half as well: both of the last two products may be done before anybody asks.)
enum Barrier {
    kQFull = 0, kSFull = 2, kPFull = 6, kODone = 10, kJobFull = 14, kJobEmpty = 16, kKFull = 18, kKEmpty = 21, kVFull = 24, kVEmpty = 27,
    kKCodesFull = 30, kKCodesEmpty = 33, kVCodesFull = 36, kVCodesEmpty = 39,
    kHalfDone = 42, kClosed = 44, kAllLeft = 46, kBarriers = 47
};

__device__ __forceinline__ int arrivals(int bar)
{
    if (bar < kSFull) return 4;                                // warps of a half
    if (bar < kPFull) return 1;                                // commits
    if (bar < kODone) return 4;
    if (bar < kJobEmpty) return 1;
    if (bar < kKFull) return kWorkers;
    if (bar < kKEmpty) return 4;
    if (bar < kVFull) return 2;                                // halves
    if (bar < kVEmpty) return 4;
    if (bar < kKCodesFull) return 2;
    if (bar < kKCodesEmpty) return 1;
    if (bar < kVCodesFull) return 4;
    if (bar < kVCodesEmpty) return 1;
    if (bar < kClosed) return 4;                               // warps of a converting group, and of a half
    return bar < kAllLeft ? 1 : kWorkers;
}

__device__ __forceinline__ uint32_t smem_address(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

// One arrival for the warp, behind what all its lanes have done. (An arrival per lane is 32 atomic operations one after another.)
__device__ __forceinline__ void arrive(uint64_t *bar)
{
    __syncwarp();
    if ((threadIdx.x & 31) == 0)
        asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_address(bar)) : "memory");
}

// What a wait needs to give up: a word of the CTA that says whether one has, and the longest time in nanoseconds.
struct Patience {
    volatile int *given_up;
    uint32_t limit;
};

__device__ __forceinline__ uint32_t nanoseconds()
{
    uint32_t t;
    asm volatile("mov.u32 %0, %%globaltimer_lo;" : "=r"(t));
    return t;
}

// One look for the phase with parity `parity`, sleeping until it comes or up to `sleep` nanoseconds.
__device__ __forceinline__ bool has_come(uint32_t at, uint32_t parity, uint32_t sleep)
{
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done) : "r"(at), "r"(parity), "r"(sleep) : "memory");
    return done != 0;
}

// Waits for the phase with parity `parity`; false where it has not come when the CTA gives up.
__device__ __forceinline__ bool wait(uint64_t *bar, uint32_t parity, const Patience &p)
{
#pragma unroll 1
    while (!has_come(smem_address(bar), parity, kSleep))
        if (*p.given_up) return false;
    return true;
}

// The same for a warp of the two that fetch codes, which looks at the clock meanwhile: where the phase does not come in time, the CTA gives up.
// (In every wait the clock costs the working warps 3 % of the kernel's time.) Whatever stops, one of these two waits for it before long.
__device__ __forceinline__ bool timed_wait(uint64_t *bar, uint32_t parity, const Patience &p)
{
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done) : "r"(smem_address(bar)), "r"(parity) : "memory");
    bool here = done != 0;
    const uint32_t began = nanoseconds();
    while (!here && !*p.given_up) {
        if (nanoseconds() - began >= p.limit) *p.given_up = 1;
        else here = has_come(smem_address(bar), parity, min(p.limit, kSleep));
    }
    // (also where the phase has come: what is given back after giving up may not have arrived yet)
    return __all_sync(0xffffffffu, here && !*p.given_up);
}

// For what must not be left behind when the CTA ends: a second at most, whatever the others have given up.
__device__ __forceinline__ void wait_for_own(uint64_t *bar, uint32_t parity)
{
    const uint32_t began = nanoseconds();
#pragma unroll 1
    while (!has_come(smem_address(bar), parity, kSleep) && nanoseconds() - began < 1000000000u) {}
}

// `bytes` of global memory to shared memory; their arrival counts for the barrier.
__device__ __forceinline__ void bulk_load(uint32_t to, const void *from, uint32_t bytes, uint64_t *bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(to), "l"(from), "r"(bytes), "r"(smem_address(bar)) : "memory");
}

__device__ __forceinline__ void arrive_expecting(uint64_t *bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_address(bar)), "r"(bytes) : "memory");
}

__device__ __forceinline__ bool elected()
{
    uint32_t yes;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
    return yes != 0;
}

// Shared memory operand in the 128-byte swizzle. `leading`, `stride`: bytes between blocks of 64 elements along the contiguous dimension
// (where that is not the one summed over) and between groups of 8 rows.
__device__ __forceinline__ uint64_t descriptor(uint32_t address, uint32_t leading, uint32_t stride)
{
    return (uint64_t)((address & 0x3ffffu) >> 4) | (uint64_t)(leading >> 4) << 16 | (uint64_t)(stride >> 4) << 32 | 1ull << 46 | 2ull << 61;
}

// fp16 operands, fp32 accumulator, M = 128; B with its N dimension contiguous if `n_major`.
__device__ __forceinline__ constexpr uint32_t instruction(int n, bool n_major)
{
    return 1u << 4 | (n_major ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (uint32_t)(128 >> 4) << 24;
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}

__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}

__device__ __forceinline__ void commit(uint64_t *bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_address(bar)) : "memory");
}

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

#define MACKO_R8(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3]), "=r"(v[i + 4]), "=r"(v[i + 5]), "=r"(v[i + 6]), "=r"(v[i + 7])
#define MACKO_W8(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3]), "r"(v[i + 4]), "r"(v[i + 5]), "r"(v[i + 6]), "r"(v[i + 7])

// 32 columns of tensor memory for the warp's 32 lanes, one lane per thread. Complete when it returns.
__device__ __forceinline__ void tmem_load32(uint32_t address, uint32_t *v)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
                 "%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
                 : MACKO_R8(v, 0), MACKO_R8(v, 8), MACKO_R8(v, 16), MACKO_R8(v, 24) : "r"(address) : "memory");
}

__device__ __forceinline__ void tmem_load64(uint32_t address, uint32_t *v)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
                 "%24,%25,%26,%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,"
                 "%56,%57,%58,%59,%60,%61,%62,%63}, [%64];\n\ttcgen05.wait::ld.sync.aligned;"
                 : MACKO_R8(v, 0), MACKO_R8(v, 8), MACKO_R8(v, 16), MACKO_R8(v, 24), MACKO_R8(v, 32), MACKO_R8(v, 40), MACKO_R8(v, 48), MACKO_R8(v, 56)
                 : "r"(address) : "memory");
}

__device__ __forceinline__ void tmem_store32(uint32_t address, const uint32_t *v)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
                 "%24,%25,%26,%27,%28,%29,%30,%31};"
                 ::MACKO_W8(v, 0), MACKO_W8(v, 8), MACKO_W8(v, 16), MACKO_W8(v, 24), "r"(address) : "memory");
}

__device__ __forceinline__ void tmem_store16(uint32_t address, const uint32_t *v)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
                 ::MACKO_W8(v, 0), MACKO_W8(v, 8), "r"(address) : "memory");
}

__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Two fp32 values in one register pair.
__device__ __forceinline__ uint64_t pair(float lo, float hi)
{
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}

__device__ __forceinline__ float2 unpair(uint64_t v)
{
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
}

__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}

__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b)
{
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

__device__ __forceinline__ float max3(float a, float b, float c)
{
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Tiles of a unit that each half of its rows takes part in, cut to a piece: [first, end[h]); rows[h] is 0 for a half without rows.
struct HalfTiles {
    int first, end[2], rows[2], last;   // last: the later end
};

__device__ __forceinline__ HalfTiles half_tiles(const AttentionArgs &a, const UnitRows &u, const Piece &p)
{
    HalfTiles h;
    h.first = p.first_tile;
    const int n = u.rows();
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        h.rows[w] = min(max(n - 128 * w, 0), 128);
        const int last_query = (128 * w + h.rows[w] - 1) / u.heads;
        const int seen = h.rows[w] > 0 ? max(0, min(u.begin + last_query + 1, a.rows.capacity)) : 0;
        h.end[w] = min((seen + kTile - 1) / kTile, p.first_tile + p.tiles);
    }
    h.last = max(h.end[0], h.end[1]);
    return h;
}

// A piece as the working warps are given it: by one warp that does nothing else, through two slots of shared memory. (Finding it
// takes 64-bit divisions: as a part of every role it made the kernel three times as long, and the roles waited for their instructions.)
struct Job {
    UnitRows u;
    HalfTiles h;             // first < 0: there are no more
    int sequence, kv_head, pieces;
    bool begins, ends;
};

__device__ __forceinline__ bool next_job(Job &job, const Job *jobs, uint64_t *bars, int &count, const Patience &patience)
{
    const int slot = count & 1;
    // a warp goes on or leaves as a whole
    if (!__all_sync(0xffffffffu, wait(bars + kJobFull + slot, (count >> 1) & 1, patience))) return false;
    job = jobs[slot];
    arrive(bars + kJobEmpty + slot);
    ++count;
    return job.h.first >= 0;
}

// Finds the next piece and gives it to the others, and to the caller.
__device__ __forceinline__ bool publish_job(Job &job, Job *jobs, WorkWalk &walk, const AttentionArgs &a, uint64_t *bars, int &count, const Patience &patience)
{
    Piece piece;
    const bool more = walk.next(a.work, a.rows, piece);
    job.h.first = -1;
    if (more) {
        job.u = unit_rows(a, walk.s, piece);
        job.h = half_tiles(a, job.u, piece);
        job.sequence = piece.sequence;
        job.kv_head = piece.kv_head;
        job.pieces = piece.pieces;
        job.begins = piece.begins;
        job.ends = piece.ends;
    }
    const int slot = count & 1;
    if (!timed_wait(bars + kJobEmpty + slot, ((count >> 1) & 1) ^ 1, patience)) return false;
    if ((threadIdx.x & 31) == 0) jobs[slot] = job;
    arrive(bars + kJobFull + slot);
    ++count;
    return more;
}

template <bool BF16, bool E4M3, int D>
__global__ void __launch_bounds__(kThreads, 1)
prompt_kernel(const AttentionArgs a)
{
    using L = Layout<D>;
    constexpr int kStages = L::kStages;
    constexpr uint32_t kQBlock = 128 * 128, kBlock = kTile * 128;   // 64 dimensions of Q, and of K or V
    extern __shared__ uint8_t raw[];
    __shared__ __align__(8) uint64_t bars[kBarriers];
    // of 16 tokens: scale of the keys, log2 and inverse of the values'. A scale that is not finite becomes (0, 1e30, NaN): a row that
    // sees a token of such a page has a sum of NaN, and one that does not has nothing of it
    __shared__ float4 scales[kConstSlots][kGroups];
    __shared__ uint32_t tmem_base;
    __shared__ int present[2][kConstSlots];           // of a tile of keys and of values: which of its blocks of 16 tokens lie on a page
    __shared__ Job jobs[2];
    __shared__ int given_up_word;
    const Patience patience = {&given_up_word, a.wait_limit};
    uint8_t *smem = raw + ((1024u - (smem_address(raw) & 1023u)) & 1023u);
    const RowsView &r = a.rows;
    const CacheView &c = a.cache;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, group = tid >> 7;

    asm volatile("griddepcontrol.launch_dependents;");
    if (tid == 0) {
        given_up_word = 0;
        for (int i = 0; i < kBarriers; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_address(bars + i)), "r"(arrivals(i)));
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_address(&tmem_base)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (tid == 0) a.split[blockIdx.x].pieces = a.split[blockIdx.x].lost = 0;
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_base;   // columns: two S of 64 of half 0 and of half 1, O of the halves (D each)
    Job job;
    int job_count = 0;

    if (group < 2) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
        const int half = group, local = tid & 127;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;
        const uint32_t s_half = tmem + lanes + half * 128, o_at = tmem + lanes + 256 + half * D;
        int done = 0;                       // tiles of this half in the pieces before
        int slot0 = 0;                      // tiles of the pieces before: where this piece's scales begin
        while (next_job(job, jobs, bars, job_count, patience)) {
            const UnitRows &u = job.u;
            const HalfTiles &h = job.h;
            if (h.rows[half] > 0) {
                const int row = half * 128 + local, query = row / u.heads, head = u.head + row % u.heads;
                const bool there = local < h.rows[half];
                float factor = fabsf(a.scale);
                if (h.first < h.end[half]) {
                    // this half of Q, as fp16, with the sign of the scale: a warp its own 32 rows, some lanes a row
                    constexpr int kLanes = D / 8, kRows = 32 / kLanes;   // lanes of a row, rows at a time
                    const int chunk = lane % kLanes;
                    const long long own_at = (long long)(u.first_row + query) * a.q_row_stride + (long long)head * a.q_head_stride;
                    uint8_t *to = smem + L::kQ + half * L::kHalf + (chunk >> 3) * kQBlock;
                    float own_up = 1.f;
                    constexpr int kBatch = 8;                            // loads under way
#pragma unroll 1
                    for (int b = 0; b < 32 / kRows; b += kBatch) {
                        uint4 q[kBatch];
#pragma unroll
                        for (int i = 0; i < kBatch; ++i) {
                            const int from = (b + i) * kRows + lane / kLanes;
                            const long long at = __shfl_sync(0xffffffffu, own_at, from);
                            load_if(q[i], a.q + at + 8 * chunk, (local & ~31) + from < h.rows[half]);
                        }
#pragma unroll
                        for (int i = 0; i < kBatch; ++i) {
                            const int row_at = (local & ~31) + (b + i) * kRows + lane / kLanes;
                            uint32_t *x = &q[i].x;
                            if (BF16) {
                                float most = 0.f, down, up;
#pragma unroll
                                for (int k = 0; k < 4; ++k) {
                                    const float2 f = unpack2<true>(x[k]);
                                    most = fmaxf(most, fmaxf(fabsf(f.x), fabsf(f.y)));
                                }
#pragma unroll
                                for (int o = 1; o < kLanes; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                                row_power(most, down, up);
#pragma unroll
                                for (int k = 0; k < 4; ++k) {
                                    const float2 f = unpack2<true>(x[k]);
                                    x[k] = pack2<false>(f.x * down, f.y * down);
                                }
                                up = __shfl_sync(0xffffffffu, up, (lane % kRows) * kLanes);
                                if (lane / kRows == b + i) own_up = up;
                            }
                            if (a.scale < 0.f) {
#pragma unroll
                                for (int k = 0; k < 4; ++k) x[k] ^= 0x80008000u;
                            }
                            *reinterpret_cast<uint4 *>(to + row_at * 128 + (((chunk & 7) ^ (row_at & 7)) << 4)) = q[i];
                        }
                    }
                    factor *= own_up;
                    fence_shared();
                    arrive(bars + kQFull + half);
                }
                const int limit = there ? min(u.begin + query + 1, r.capacity) : 0;           // tokens that this row sees
                const int all_see = min(u.begin + 128 * half / u.heads + 1, r.capacity);      // that every row of this half sees
                float m = -INFINITY, l = 0.f;
                bool far = false;   // a row of the warp has a maximum from 2^20 on
#pragma unroll 1
                for (int j = h.first; j < h.end[half]; ++j) {
                    const int count = done + j - h.first, buffer = count & 1;
                    const uint32_t s_at = s_half + 64 * buffer;
                    const bool late = !wait(bars + kSFull + 2 * half + buffer, (count >> 1) & 1, patience);
                    __syncwarp();
                    fence_after();
                    const float4 *of_tile = scales[(slot0 + j - h.first) % kConstSlots];
                    float s[kTile], most = -INFINITY;
                    tmem_load64(s_at, reinterpret_cast<uint32_t *>(s));
                    if ((j + 1) * kTile > all_see) {
                        const int see = limit - j * kTile;
#pragma unroll
                        for (int i = 0; i < kTile; ++i) s[i] = i < see ? s[i] : -INFINITY;
                    }
#pragma unroll
                    for (int g = 0; g < kGroups; ++g) {
                        const float4 k = of_tile[g];
                        const float *x = s + 16 * g;
                        float top = max3(x[0], x[1], x[2]), top2 = max3(x[3], x[4], x[5]);
                        top = max3(top, x[6], x[7]);
                        top2 = max3(top2, x[8], x[9]);
                        top = max3(top, x[10], x[11]);
                        top2 = max3(top2, x[12], x[13]);
                        top = max3(top, x[14], x[15]);
                        most = fmaxf(most, fmaf(fmaxf(top, top2), fmaxf(k.x * factor, kLeastFactor), k.y));
                    }
                    const bool grown = most - m > kTop;   // the difference of numbers that are near one another is exact
                    if (__any_sync(0xffffffffu, grown || late)) {
                        if (__any_sync(0xffffffffu, late)) break;   // given up
                        const float to = grown ? __fadd_ru(most, kLag - kTop) : m, keep = grown ? exp2_fast(m - to) : 1.f;
                        m = to;
                        far = __any_sync(0xffffffffu, m > kFar || (m < -kFar && m > -INFINITY));
                        l *= keep;
                        if (j > h.first) {
                            wait(bars + kODone + 2 * half + (buffer ^ 1), ((count - 1) >> 1) & 1, patience);
                            __syncwarp();
                            fence_after();
#pragma unroll 1
                            for (int i = 0; i < D; i += 32) {
                                uint32_t o[32];
                                tmem_load32(o_at + i, o);
#pragma unroll
                                for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * keep);
                                tmem_store32(o_at + i, o);
                            }
                            tmem_store_wait();
                        }
                    }
                    const float base = m == -INFINITY ? 0.f : m;
                    // 2^x below takes the product's own rounding and that of k.y - base for nothing, which holds as long as fp32 has fractions of the
                    // maximum. Beyond, x is what the maximum was found from, less m: nothing is above 2^15 then either.
                    if (__builtin_expect(far, 0)) {
#pragma unroll
                        for (int i = 0; i < kTile; ++i) {
                            const float4 k = of_tile[i / 16];
                            s[i] = fmaf(s[i], fmaxf(k.x * factor, kLeastFactor), k.y) - base;
                        }
                    }
#pragma unroll
                    for (int two = 0; two < 2; ++two) {
                        uint32_t p[16];
#pragma unroll
                        for (int gg = 0; gg < 2; ++gg) {
                            const int g = 2 * two + gg;
                            const float4 k = of_tile[g];
                            const float by = far ? 1.f : fmaxf(k.x * factor, kLeastFactor), plus = far ? 0.f : k.y - base;
                            const uint64_t by2 = pair(by, by), plus2 = pair(plus, plus);
                            uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
                            for (int i = 0; i < 16; i += 2) {
                                const float2 x = unpair(fma_pair(pair(s[16 * g + i], s[16 * g + i + 1]), by2, plus2));
                                const float e0 = exp2_fast(x.x), e1 = exp2_fast(x.y);
                                sum[(i >> 1) & 1] = add_pair(sum[(i >> 1) & 1], pair(e0, e1));
                                p[8 * gg + i / 2] = pack2<false>(e0, e1);
                            }
                            const float2 both = unpair(add_pair(sum[0], sum[1]));
                            const float all = both.x + both.y;
                            l += all == 0.f ? 0.f : all * k.z;   // tokens that a row does not see may have any scale
                        }
                        tmem_store16(s_at + 16 * two, p);
                    }
                    tmem_store_wait();
                    fence_before();
                    arrive(bars + kPFull + 2 * half + buffer);
                }
                // the result of this half, divided or as a piece
                if (h.first < h.end[half]) {
                    done += h.end[half] - h.first;
                    wait(bars + kODone + 2 * half + ((done - 1) & 1), ((done - 1) >> 1) & 1, patience);
                    __syncwarp();
                    fence_after();
                }
                const bool alone = job.begins && job.ends, empty = h.first >= h.end[half];
                float *partial = a.partial + ((long long)blockIdx.x * 2 + (job.begins ? 1 : 0)) * L::kRows * (D + 2);
                const float by = alone ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
                // through this half's place for Q, which the tensor core is done with, so that some lanes write a row: 16-bit values in
                // one pass, fp32 in two
                const long long own_to = alone ? ((long long)(u.first_row + query) * a.heads + head) * D : (long long)row * D;
                uint8_t *mine = smem + L::kQ + half * L::kHalf + (local >> 5) * (L::kHalf / 4);
#pragma unroll 1
                for (int pass = 0; pass < (alone ? 1 : 2); ++pass) {
                    __syncwarp();
#pragma unroll 1
                    for (int i = 0; i < (alone ? D : D / 2); i += 32) {
                        uint32_t o[32];
                        if (!empty) {
                            tmem_load32(o_at + pass * (D / 2) + i, o);
                        } else {
#pragma unroll
                            for (int k = 0; k < 32; ++k) o[k] = 0u;
                        }
                        uint8_t *at = mine + lane * (2 * D);
                        if (alone) {
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                uint4 v;
#pragma unroll
                                for (int n = 0; n < 4; ++n)
                                    (&v.x)[n] = pack2<BF16>(__uint_as_float(o[8 * k + 2 * n]) * by, __uint_as_float(o[8 * k + 2 * n + 1]) * by);
                                *reinterpret_cast<uint4 *>(at + (((i / 8 + k) ^ (lane & 7)) << 4)) = v;
                            }
                        } else {
#pragma unroll
                            for (int k = 0; k < 8; ++k)
                                *reinterpret_cast<float4 *>(at + (((i / 4 + k) ^ (lane & 7)) << 4)) =
                                    make_float4(__uint_as_float(o[4 * k]) * by, __uint_as_float(o[4 * k + 1]) * by, __uint_as_float(o[4 * k + 2]) * by,
                                                __uint_as_float(o[4 * k + 3]) * by);
                        }
                    }
                    __syncwarp();
                    constexpr int kLanes = D / 8, kRows = 32 / kLanes;
                    const int chunk = lane % kLanes;
#pragma unroll 4
                    for (int i = 0; i < 32; i += kRows) {
                        const int from = i + lane / kLanes;
                        const long long to = __shfl_sync(0xffffffffu, own_to, from);
                        const uint4 v = *reinterpret_cast<const uint4 *>(mine + from * (2 * D) + ((chunk ^ (from & 7)) << 4));
                        if ((local & ~31) + from >= h.rows[half]) continue;
                        if (alone) reinterpret_cast<uint4 *>(a.out + to)[chunk] = v;
                        else reinterpret_cast<uint4 *>(partial + to + pass * (D / 2))[chunk] = v;
                    }
                }
                if (there && !alone) {
                    partial[L::kRows * D + row] = m;
                    partial[L::kRows * D + L::kRows + row] = l;
                }
                if (!alone && job.begins && row == 0)
                    a.split[blockIdx.x] = SplitUnit{u.first_row, u.rows(), u.head, job.pieces, u.heads, 0, {0, 0}};
                fence_before();   // O is read before this half arrives for the next piece's P
            }
            // nobody's part of Q is written while another warp still has results there
            arrive(bars + kHalfDone + half);
            wait(bars + kHalfDone + half, (job_count - 1) & 1, patience);
            __syncwarp();
            slot0 += max(h.last - h.first, 0);
        }
    } else if (group < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        // Eight neighbouring threads take 16 codes each of two rows: of one the first 64 of 128 dimensions, of the other the last (at
        // head_dim 64: all of both), so that what they read and both 16-byte pieces of what they write lie in different banks.
        const bool is_v = group == 3;
        constexpr int kItems = kTile * D / 16 / 128;     // that a thread converts
        constexpr int kApart = D == 64 ? 32 : D == 128 ? 16 : 8;        // rows between them
        const int local = tid & 127, eight = local & 7;
        const int row = 2 * (local >> (D == 64 ? 3 : D == 128 ? 4 : 5)) + (eight >> 2);
        const int chunk = D == 64 ? eight & 3 : (eight ^ (((local >> 3) & 1) << 2)) + (D == 256 ? ((local >> 4) & 1) * 8 : 0);
        uint64_t *full = bars + (is_v ? kVFull : kKFull), *empty = bars + (is_v ? kVEmpty : kKEmpty);
        uint64_t *codes_full = bars + (is_v ? kVCodesFull : kKCodesFull), *codes_empty = bars + (is_v ? kVCodesEmpty : kKCodesEmpty);
        const uint8_t *const from = smem + (is_v ? L::kVCodes : L::kKCodes) + row * D + chunk * 16;
        uint8_t *const to = smem + (is_v ? L::kV : L::kK) + (chunk >> 2) * kBlock + row * 128;
        const int lo_at = ((2 * (chunk & 3)) ^ (row & 7)) << 4, hi_at = lo_at ^ 16;
        int n = 0;                                       // tiles so far
        Ring<L::kStages> ring;
        Ring<L::kCodeStages> codes_ring;
        while (next_job(job, jobs, bars, job_count, patience)) {
            const HalfTiles &h = job.h;
            const int end = max(0, min(job.u.begin + job.u.queries, r.capacity));   // no row sees anything from here on
#pragma unroll 1
            for (int j = h.first; j < h.last; ++j, ++n) {
                if (!__all_sync(0xffffffffu, wait(codes_full + codes_ring.stage, codes_ring.phase, patience) && wait(empty + ring.stage, ring.phase ^ 1u, patience)))
                    break;
                const int blocks = present[is_v][n % kConstSlots];
                const int rows = blocks == (1 << kGroups) - 1 ? end - j * kTile : -1;   // that are there, if all pages are
#pragma unroll
                for (int i = 0; i < kItems; ++i) {
                    uint4 x = *reinterpret_cast<const uint4 *>(from + codes_ring.stage * L::kCodes + i * kApart * D), lo, hi;
                    if (rows < kTile) {   // the same for all threads: nothing behind the last token and on pages that are none may be NaN
                        const int at = row + i * kApart;
                        if (!(blocks >> (at >> 4) & 1) || j * kTile + at >= end) x = make_uint4(0u, 0u, 0u, 0u);
                    }
                    codes_to_half<E4M3>(x.x, lo.x, lo.y);
                    codes_to_half<E4M3>(x.y, lo.z, lo.w);
                    codes_to_half<E4M3>(x.z, hi.x, hi.y);
                    codes_to_half<E4M3>(x.w, hi.z, hi.w);
                    *reinterpret_cast<uint4 *>(to + ring.stage * L::kStage + i * kApart * 128 + lo_at) = lo;
                    *reinterpret_cast<uint4 *>(to + ring.stage * L::kStage + i * kApart * 128 + hi_at) = hi;
                }
                fence_shared();
                arrive(codes_empty + codes_ring.stage);
                arrive(full + ring.stage);
                ring.next();
                codes_ring.next();
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
        if (warp < 18) {
            // One half's products. The whole warp walks and waits; one elected thread issues. What the instructions take is the same in all
            // lanes in a way that the compiler can see (shuffles, election), so that it stays in uniform registers: with `if (lane == 0)`
            // an issue took some 200 cycles. Each half has a warp of its own because a wait for what is there already takes some 150.
            const int w = warp - 16;
            const uint32_t d_at = __shfl_sync(0xffffffffu, tmem, 0), operands = __shfl_sync(0xffffffffu, smem_address(smem), 0);
            const uint32_t o = d_at + 256 + w * D;
            const uint64_t q = descriptor(operands + L::kQ + w * L::kHalf, 16, 1024);
            int n = 0, done = 0;                  // tiles of the pieces before, and those of them that this half took part in
            uint32_t q_phase = 0;
            while (next_job(job, jobs, bars, job_count, patience)) {
                const int first = __shfl_sync(0xffffffffu, job.h.first, 0), end = __shfl_sync(0xffffffffu, w ? job.h.end[1] : job.h.end[0], 0);
                const int last = __shfl_sync(0xffffffffu, job.h.last, 0);
                // S of the first two tiles, then for every tile: O += P V, and S of the second tile behind it. Tiles that the other half
                // alone takes part in are let go as they come.
#pragma unroll 1
                for (int j = first - 2; j < last; ++j) {
                    const int tile = n + j - first, count = done + j - first;
                    const uint32_t s = d_at + 128 * w + 64 * (count & 1);   // of this tile and of the second one behind it
                    if (j >= first) {
                        const unsigned use = (unsigned)tile / kStages;
                        const int stage = tile - use * kStages;
                        wait(bars + kVFull + stage, use & 1, patience);
                        if (j < end) {
                            if (!__all_sync(0xffffffffu, wait(bars + kPFull + 2 * w + (count & 1), (count >> 1) & 1, patience))) break;
                            fence_after();
                            if (elected()) {
                                const uint64_t v = descriptor(operands + L::kV + stage * L::kStage, kBlock, 1024);
#pragma unroll
                                for (int t = 0; t < kTile / 16; ++t) mma_ts(o, s + 8 * t, v + t * (2048 >> 4), instruction(D, true), j > first || t > 0);
                                commit(bars + kODone + 2 * w + (count & 1));
                                commit(bars + kVEmpty + stage);
                            }
                            __syncwarp();
                        } else {
                            arrive(bars + kVEmpty + stage);
                        }
                    }
                    if (j + 2 < last) {
                        const unsigned use = (unsigned)(tile + 2) / kStages;
                        const int stage = tile + 2 - use * kStages;
                        wait(bars + kKFull + stage, use & 1, patience);
                        if (j + 2 < end) {
                            if (j + 2 == first) {
                                wait(bars + kQFull + w, q_phase, patience);
                                q_phase ^= 1u;
                            }
                            __syncwarp();
                            fence_after();
                            if (elected()) {
                                const uint64_t k = descriptor(operands + L::kK + stage * L::kStage, 16, 1024);
#pragma unroll
                                for (int d = 0; d < D / 16; ++d)
                                    mma_ss(s, q + (((d >> 2) * kQBlock + (d & 3) * 32) >> 4), k + (((d >> 2) * kBlock + (d & 3) * 32) >> 4),
                                           instruction(kTile, false), d > 0);
                                commit(bars + kSFull + 2 * w + (count & 1));
                                commit(bars + kKEmpty + stage);
                            }
                            __syncwarp();
                        } else {
                            arrive(bars + kKEmpty + stage);
                        }
                    }
                }
                n += max(last - first, 0);
                done += max(end - first, 0);
            }
            // all that was issued has arrived before shared and tensor memory are given back
            if (elected()) commit(bars + kClosed + w);
            __syncwarp();
            wait_for_own(bars + kClosed + w, 0);
            __syncwarp();
        } else {
            // codes of keys (warp 18, with the scales of both) or of values: one lane for each block of 16 tokens, eight tiles at a time
            const bool is_v = warp == 19;
            uint64_t *full = bars + (is_v ? kVCodesFull : kKCodesFull), *empty = bars + (is_v ? kVCodesEmpty : kKCodesEmpty);
            const uint32_t codes = smem_address(smem + (is_v ? L::kVCodes : L::kKCodes));
            const int page_mask = (1 << c.page_log2) - 1, own_tile = lane / kGroups, block = lane % kGroups;
            int n = 0;
            Ring<L::kCodeStages> ring;
            WorkWalk walk;
            bool came = true;
            if (!is_v) walk.start(a.work, r, blockIdx.x);
            asm volatile("fence.proxy.async.global;" ::: "memory");   // the cache may have been written by the kernel in front
            while (came && (is_v ? next_job(job, jobs, bars, job_count, patience) : publish_job(job, jobs, walk, a, bars, job_count, patience))) {
                const HalfTiles &h = job.h;
                const int end = max(0, min(job.u.begin + job.u.queries, r.capacity));
                const uint8_t *base = (is_v ? c.v : c.k) + ((long long)job.kv_head << c.page_log2) * D;
                const long long page_stride = is_v ? c.v_stride : c.k_stride;
#pragma unroll 1
                for (int j0 = h.first; j0 < h.last && came; j0 += 32 / kGroups) {
                    const int tile = j0 + own_tile, token = tile * kTile + 16 * block;
                    const int page = tile < h.last && token < end ? page_at(c, r, job.sequence, token) : -1;
                    const uint8_t *source = base + page * page_stride + (token & page_mask) * D;
                    float4 of_lane = make_float4(0.f, -INFINITY, 0.f, 0.f);
                    if (!is_v && page >= 0) {
                        const float ks = __ldcg(c.k_scale + page * c.k_scale_stride + job.kv_head);
                        const float vs = value_scale(__ldcg(c.v_scale + page * c.v_scale_stride + job.kv_head));
                        of_lane = ks < INFINITY && vs < INFINITY ? make_float4(ks, __log2f(vs), inverse_scale(vs), 0.f)
                                                                 : make_float4(0.f, 1e30f, __uint_as_float(0x7fffffffu), 0.f);
                    }
                    // with one stage of codes the way from memory would be a part of every tile: from the L2 cache it is a short one
                    if (L::kCodeStages == 1 && page >= 0)
                        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(source), "r"(16 * D) : "memory");
                    const uint32_t all = __ballot_sync(0xffffffffu, page >= 0);
#pragma unroll 1
                    for (int t = 0; t < 32 / kGroups && j0 + t < h.last; ++t, ++n) {
                        came = timed_wait(empty + ring.stage, ring.phase ^ 1u, patience);
                        if (!came) break;
                        const int blocks = (all >> (t * kGroups)) & ((1 << kGroups) - 1);
                        if (lane == 0) present[is_v][n % kConstSlots] = blocks;
                        if (!is_v && own_tile == t) scales[n % kConstSlots][block] = of_lane;
                        __syncwarp();
                        if (lane == 0) arrive_expecting(full + ring.stage, __popc(blocks) * 16 * D);
                        __syncwarp();
                        if (own_tile == t && page >= 0) bulk_load(codes + ring.stage * L::kCodes + block * 16 * D, source, 16 * D, full + ring.stage);
                        ring.next();
                    }
                }
            }
            // no copy is in flight when the CTA's shared memory is given back
            for (int k = max(n - L::kCodeStages, 0); k < n; ++k) wait_for_own(full + k % L::kCodeStages, (k / L::kCodeStages) & 1);
            __syncwarp();
            const bool all_left = is_v || timed_wait(bars + kAllLeft, 0, patience);
            if (!is_v && __any_sync(0xffffffffu, !all_left || *patience.given_up)) {
                // given up: NaN for all rows that the CTA has a part in, when nobody else writes any more
                wait_for_own(bars + kAllLeft, 0);
                Piece piece;
                walk.start(a.work, r, blockIdx.x);
                while (walk.next(a.work, r, piece)) {
                    const UnitRows u = unit_rows(a, walk.s, piece);
                    for (int row = 0; row < u.rows(); ++row) {
                        uint32_t *to = reinterpret_cast<uint32_t *>(a.out + ((long long)(u.first_row + row / u.heads) * a.heads + u.head + row % u.heads) * D);
                        for (int i = lane; i < D / 2; i += 32) to[i] = 0x7fff7fffu;
                    }
                }
                if (lane == 0) a.split[blockIdx.x].lost = 1;
            }
        }
    }
    if (warp != 18) arrive(bars + kAllLeft);
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == 16) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    clear_other_rows(a);
}

template <bool BF16, bool E4M3, int D>
int launch(const AttentionArgs &a, cudaStream_t stream)
{
    static bool raised[kMaxDevices];   // dynamic shared memory above 48 KB is allowed per kernel and device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev >= kMaxDevices || !raised[dev])) {
        e = cudaFuncSetAttribute(prompt_kernel<BF16, E4M3, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<D>::kBytes);
        if (e == cudaSuccess && dev < kMaxDevices) raised[dev] = true;
    }
    if (e != cudaSuccess) return fail(MACKO_ERR_CUDA, "paged_attention: %s", cudaGetErrorString(e));
    return launch_pdl("paged_attention", prompt_kernel<BF16, E4M3, D>, dim3(a.work.ctas), dim3(kThreads), 1, Layout<D>::kBytes, stream, a);
}

template <int D>
int launch_types(const AttentionArgs &a, bool bf16, bool e4m3, cudaStream_t s)
{
    if (bf16) return e4m3 ? launch<true, true, D>(a, s) : launch<true, false, D>(a, s);
    return e4m3 ? launch<false, true, D>(a, s) : launch<false, false, D>(a, s);
}

}  // namespace

int launch_prompt_attention(const AttentionArgs &a, bool bf16, bool e4m3, cudaStream_t stream)
{
    switch (a.cache.head_dim) {
    case 64: return launch_types<64>(a, bf16, e4m3, stream);
    case 128: return launch_types<128>(a, bf16, e4m3, stream);
    default: return launch_types<256>(a, bf16, e4m3, stream);
    }
}

}  // namespace macko
