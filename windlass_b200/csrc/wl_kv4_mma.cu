// Attention of prompts over the 4-bit KV cache on the 5th-generation tensor cores (tcgen05, sm_100a).
//
// A CTA takes 128 queries ((row, head) pairs of a run of rows that share a cache) of one KV head and walks the visible
// positions in steps of 128 (8 cache tiles). Scores and output are tcgen05 products with fp32 sums in tensor memory:
//   S[128 queries][128 positions] = Q K',    O[128 queries][HD] += P V'.
// Everything enters as two fp16 planes, a value's rounding and what it left: Q (scaled by a power of two a row) and the
// weights P 22 bits, K' = (c - 8) d and V' = (c - 8) d vs exactly (a 4-bit code times an 11-bit scale has at most 15 bits; vs
// is a power of two, 2^8 unless a step has a value scale of 2 or more). Only in a step with a key scale of 2^13 or more, whose
// products would pass fp16's largest, is K' (c - 8) d 2^-3; key scales below 2^-11 beside it lose bits, and so do value scales
// below 2^-14 / vs: less than 2^-22 of the step's largest, both.
// A query's weights of a step are scaled by a power of two of their own that brings the step's largest to 2^14..2^15: fp16
// has no steps below 2^-24, so beside weights left as they are, at most 1, one of 2^-25 would be lost, and of a few
// thousand positions 12 nats below a sink the output lost 2e-3. So scaled, weights keep 22 bits down to 2^-16 of their
// step's largest, and what is lost below is at most 2^-39 of it.
// Each product is three MMAs, hi hi + lo hi + hi lo; the dropped lo lo is below 2^-22 of it, so the result is as exact as fp32
// arithmetic. Q and P are the MMA's A operand in tensor memory (P in the place of the scores it came from), K' and V' its B
// operand in shared memory.
//   - warp 13 copies a step's cache tiles (contiguous 18 HD bytes each) into a ring of raw steps with bulk copies, warp 14
//     looks their value scales over;
//   - warps 4-11 turn codes into the planes of K' and V' in the 128-byte-swizzled K-major layout. The order of a step's
//     positions is chosen so that a thread's codes are whole 16-byte chunks of it: within 32 positions, slot 8 c + 2 (2 t + h)
//     + e is position 16 t + 8 h + 2 c + e; within 8 dims, 0 4 1 5 2 6 3 7. Both products use the same order;
//   - warp 12 issues the MMAs;
//   - warps 0-3 own a query a thread (its tensor-memory lane): maximum, weights and sum without a shuffle, and P's planes
//     back to tensor memory;
//   - warps 4-11 also keep the output in registers (32 queries by HD / 2 dims a warp): a step's product starts from zero in
//     tensor memory and is added here in fp32 (the tensor core's sums are cut off, not rounded: over 768 of them in one
//     place the output was 8e-6 off, added step by step 1e-6), scaled by what the step changed in the query's maximum.
// Order of the products: scores of step j + 1, output of step j - 1, scores of j + 2, ... with two score buffers. Tensor
// memory: scores 2 x 128 columns, the step's output 128, Q 128 (at HD = 128): all 512.
// Two blocks of queries or more go in pairs of CTAs (cta_group::2): the pair walks the positions that its 256 queries see, each
// CTA makes half of K' (64 positions) and of V' (half the dims) and the MMAs read both halves, so that a CTA unpacks half as
// much and has room for two steps of both planes. One block goes by a CTA of its own. What that gave (1500 rows of a prompt,
// 64 heads on 8 of 128 dims): 194 us by single CTAs, 195 by pairs with one step of planes, 172 with two of V' and the queries
// and outputs copied by way of shared memory (a thread's own loads of its query took 11000 cycles of a CTA's start), 162.7
// with two of K', the scales' warp and the positions' range found by each warp for itself, 160.6 with forms of their own for
// steps without masks and scales without care (less code in the instruction caches; 512 rows behind a window of 4096
// positions, 32 heads on 4: 130.7 to 108.2 us). That is 0.75 and 0.98 PFLOP/s of MMAs, of 1.65 measured. A step takes 5000 to
// 6000 cycles, of them 3700 and more of MMAs, and each other role about as long; starting and ending a CTA takes as long as 4
// or 5 steps. One thread's issue of the MMAs is close to the bound: with its loops rolled up 177 and 123 us, with
// all 48 products unrolled 159 and 111.
#include <algorithm>
#include <type_traits>
#include "wl_kv4.cuh"

namespace wl {
namespace k {

namespace {

constexpr int PM_Q = 128, PM_P = 128;       // queries of a CTA, positions of a step
constexpr int PM_TILES = PM_P / KV4_P;
constexpr int PM_RAW = 4;                   // raw steps in flight
constexpr int PM_DQ_WARP = 4, PM_DQ = 8, PM_MMA_WARP = 12, PM_RAW_WARP = 13, PM_CARE_WARP = 14, PM_THREADS = 512;
constexpr int PM_SLOTS = 8;                 // steps whose care and factors are kept
constexpr float PM_WEIGHT_BITS = 15.f;      // a step's weights are multiplied by 2^(15 - its reference maximum)
// tensor memory columns
constexpr int TM_S = 0, TM_O = 256, TM_QH = 384, TM_QL = 448;

constexpr int pm_plane(int HD) { return HD * 256; }             // one fp16 plane of a step: 128 x HD
constexpr int pm_q_row(int HD) { return HD * 4 + 16; }          // a staged query's bytes (16 more: no bank conflicts)
constexpr int pm_o_row(int HD) { return HD * 2 + 16; }          // half a staged output row's
constexpr int pm_bufs(int NC) { return NC; }                    // steps of K' and V' in shared memory: a pair's CTA has room for two
constexpr int pm_smem(int HD, int NC) { return 4 * pm_bufs(NC) * pm_plane(HD) / NC + PM_RAW * PM_TILES * kv4_tile_bytes(HD) + 1024; }

// (where the other CTA of a pair arrives)
__device__ __forceinline__ bool pm_try_wait_cluster(uint64_t* bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok;
}
// A wait bounded by time (2 s); after one gives up, all of the CTA's waits return at once.
template <bool CLUSTER = false> __device__ __forceinline__ bool pm_wait(uint64_t* bar, uint32_t parity, int* err, volatile int* abort)
{
    auto ready = [&] { return CLUSTER ? pm_try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity); };
    if (*abort) return false;
    if (ready()) return true;
    const unsigned long long t0 = globaltimer_ns();
    while (!ready()) {
        if (*abort) return false;
        if (globaltimer_ns() - t0 > MBAR_WAIT_NS) {
            atomicExch(err, 24);
            *abort = 1;
            return false;
        }
    }
    return true;
}
__device__ __forceinline__ void pm_arrive(uint64_t* bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// The same at the barrier of a pair's first CTA, which issues the MMAs.
__device__ __forceinline__ void pm_arrive_lead(uint64_t* bar)
{
    asm volatile("{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %0, 0;\n mbarrier.arrive.release.cluster.shared::cluster.b64 _, [a];\n}\n"
                 ::"r"(smem_u32(bar)) : "memory");
}
// All threads of a pair meet.
template <int NC> __device__ __forceinline__ void pm_pair_arrive()
{
    if constexpr (NC == 2) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
template <int NC> __device__ __forceinline__ void pm_pair_wait()
{
    if constexpr (NC == 2) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,"
                 "%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                   "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
                   "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
                   "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr));
}
// Waits for this thread's loads; the values of r come out of it, so that none is used before.
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[32])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                   "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]),
                   "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]),
                   "+r"(r[28]), "+r"(r[29])
                 :: "memory");
    asm volatile("" : "+r"(r[30]), "+r"(r[31]) :: "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
                 "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,"
                 "%31,%32};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
                   "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
                   "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
                   "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
                 : "memory");
}

template <int N> __device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// Shared-memory matrix descriptor: K-major, 128-byte swizzle, 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t pm_desc(const void* p)
{
    const uint64_t addr = smem_u32(p);
    return ((addr & 0x3FFFFull) >> 4) | (1ull << 16) | ((1024ull >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// kind::f16 with fp16 operands, fp32 sums, M = 128 queries a CTA.
constexpr uint32_t pm_idesc(int N, int NC) { return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(128 * NC >> 4) << 24); }

template <int NC> __device__ __forceinline__ void pm_mma(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate)
{
    if constexpr (NC == 1)
        asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                     " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
                     ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
    else
        asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                     " tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
                     ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// Arrives at the barrier (of both CTAs of a pair) when the MMAs before it are done.
template <int NC> __device__ __forceinline__ void pm_commit(uint64_t* bar)
{
    if constexpr (NC == 1)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                     ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
}

// 2^k of a whole k <= 127; 0 below 2^-126, and of -inf and NaN.
__device__ __forceinline__ float pow2i(float k) { return __int_as_float(((int)fmaxf(k, -127.f) + 127) << 23); }

// Bits [0, 16) of the positions p0 .. p0 + 15 that v sees.
__device__ __forceinline__ uint32_t seen16(const Vis& v, int p0)
{
    auto below = [&](int n) { return n <= p0 ? 0u : n >= p0 + 16 ? 0xFFFFu : (1u << (n - p0)) - 1u; };
    return below(v.n) & (~below(v.first) | below(v.sink));
}
// Those of a tile's 16 positions in the order of the step's slots: position 8 h + 2 c + e at bit 8 c + 2 h + e.
__device__ __forceinline__ uint32_t slots16(uint32_t x)
{
    auto spread = [](uint32_t y) { return (y & 3u) | (y & 0xCu) << 6 | (y & 0x30u) << 12 | (y & 0xC0u) << 18; };
    return spread(x) | spread(x >> 8) << 2;
}

// What the scales of a step call for (slot j % PM_SLOTS): whether a key's is 2^13 or more; the largest of the values' of 2 or
// more, and where those are NaN (a value row that held an infinity or NaN): bit n of word n / 32 of block b is slot n.
template <int NB> struct StepCare {
    uint32_t vmax;              // its float's bits; 0: all below 2
    int any_nan;
    int big_keys;               // K' = (c - 8) d 2^-3
    uint32_t nan[NB][PM_P / 32];
    __device__ __forceinline__ float vs() const
    {
        // V' = (c - 8) d vs stays below 2^13
        return vmax ? ldexpf(1.f, max(8 - ilogbf(__uint_as_float(vmax)), -7)) : 256.f;
    }
    __device__ __forceinline__ void clear()
    {
        vmax = 0u;
        any_nan = big_keys = 0;
        for (int b = 0; b < NB; ++b)
            for (int i = 0; i < PM_P / 32; ++i) nan[b][i] = 0u;
    }
};

template <int HD, int NC>
__global__ void __launch_bounds__(PM_THREADS, 1) k_kv4_attn_mma(const Kv4Att a, int q_blocks)
{
    constexpr int NB = HD / 32, TB = kv4_tile_bytes(HD), PL = pm_plane(HD) / NC;
    constexpr int NP = pm_bufs(NC), KP = PM_P / NC, VD = HD / NC;             // rows of K' (positions) and V' (dims) that this CTA makes
    static_assert(HD == 64 || HD == 128, "planes of whole 64-value swizzle atoms");
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t *kh = smem, *raw = smem + NP * 2 * PL, *vh = raw + PM_RAW * PM_TILES * TB;      // (each plane's remainder PL behind it)
    // the queries before the first V' and the raw steps 2 and 3; the output after the last raw step
    uint8_t *qs = raw + 2 * PM_TILES * TB, *os = raw;
    static_assert(PM_RAW == 4 && PM_Q * pm_q_row(HD) <= 2 * PM_TILES * TB + 2 * PL, "the queries end before V' does");
    static_assert(PM_DQ * 32 * pm_o_row(HD) <= PM_RAW * PM_TILES * TB && PM_RAW * PM_TILES * TB % 1024 == 0, "the output fits; V' is aligned");
    __shared__ __align__(8) uint64_t raw_full[PM_RAW], raw_empty[PM_RAW], care_full[PM_RAW], q_raw, q_read, drained, q_full, k_full[NP], v_full[NP], pv_done, o_free, s_full[2],
        p_full[2];
    __shared__ StepCare<NB> care[PM_SLOTS];
    // of a step and query: e^(old - new reference maximum), and the power of two that its weights' product is multiplied by
    __shared__ float2 factor[PM_SLOTS][PM_Q];
    __shared__ float fin_l[PM_Q];
    __shared__ uint32_t fin_poison[PM_Q];
    __shared__ uint32_t tmem_base;
    __shared__ int abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = a.heads / a.kv_heads, kvh = blockIdx.y;
    // the last queries (of a prompt: those that see most) first
    const int cta = NC == 1 ? 0 : (int)blockIdx.x % NC, group = (int)blockIdx.x / NC;
    const int qg = q_blocks / NC - 1 - group / a.S, sp = group % a.S, qb = qg * NC + cta, run = blockIdx.z;
    const int nq = a.R * G, q0 = qb * PM_Q;
    // the rows that the CTA (both CTAs) takes: each warp finds the positions that they see together (the loads are on their way
    // while the rest is set up)
    const int p0 = qg * NC * PM_Q, r0 = p0 / G, r1 = min(a.R - 1, (min(p0 + NC * PM_Q, nq) - 1) / G);
    const int pos0 = r0 + lane <= r1 ? a.pos[run * a.R + r0 + lane] : -1;
    const int qpos = warp < 4 && q0 + (int)threadIdx.x < nq ? a.pos[run * a.R + (q0 + (int)threadIdx.x) / G] : -1;
    const uint8_t* base = a.rows.base(run * a.R);
    if (warp == 2) {
        // (the first CTA of a pair counts the other's warps as one: that CTA's forwarding thread)
        const int more = NC == 2 && cta == 0;
        if (lane < PM_RAW) {
            mbar_init(&raw_full[lane], 1);
            mbar_init(&raw_empty[lane], PM_DQ);
            mbar_init(&care_full[lane], 1);
        } else if (lane < 8) {
            const int s = lane & 1;
            if (lane < 6) {
                mbar_init(&s_full[s], 1);
                mbar_init(&p_full[s], 4 + more);
            } else if (s < NP) {
                mbar_init(&k_full[s], PM_DQ + more);
                mbar_init(&v_full[s], PM_DQ);
            }
        } else if (lane == 8) {
            mbar_init(&q_raw, 4);
            mbar_init(&q_read, 4);
            mbar_init(&drained, 1);
            mbar_init(&q_full, 4);
        } else if (lane == 9) {
            mbar_init(&o_free, PM_DQ);
            mbar_init(&pv_done, 1);
            abort_flag = 0;
        }
        fence_mbar_init();
    }
    if (warp == 1 && lane < PM_SLOTS) care[lane].clear();
    if (warp == 0) {
        if constexpr (NC == 1) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)), "r"(512) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)), "r"(512) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        }
    }
    Vis seen{0, INT_MAX, 0};
    for (int r = r0 + lane; r <= r1; r += 32) {
        const int p = r < r0 + 32 ? pos0 : a.pos[run * a.R + r];
        if (kv4_row_state(base, p, a.capacity)) continue;
        const Vis v = visible(p, a.window, a.sinks);
        seen.n = max(seen.n, v.n);
        seen.first = min(seen.first, v.first);
        seen.sink = max(seen.sink, v.sink);
    }
    seen.n = __reduce_max_sync(0xffffffffu, seen.n);
    seen.first = __reduce_min_sync(0xffffffffu, seen.first);
    seen.sink = __reduce_max_sync(0xffffffffu, seen.sink);
    const TileList tl = seen.n > 0 ? tile_list(seen.n, seen.first, seen.sink) : TileList{0, 0, 0};
    int i0 = 0, i1 = tl.count;
    if (a.S > 1) {
        i0 = (int)((int64_t)tl.count * sp / a.S);
        i1 = (int)((int64_t)tl.count * (sp + 1) / a.S);
    }
    const int steps = (i1 - i0 + PM_TILES - 1) / PM_TILES;
    tc_before();
    __syncthreads();
    tc_after();
    pm_pair_arrive<NC>();                   // (this CTA's barriers and tensor memory are there)
    volatile int* abort = &abort_flag;
    auto raw_load = [&](int j) {            // (one thread) step j's cache tiles
        const int s = j % PM_RAW, at = i0 + PM_TILES * j, n = min(PM_TILES, i1 - at);
        mbar_expect_tx(&raw_full[s], n * TB);
        for (int i = 0; i < n; ++i)
            bulk_load(raw + (s * PM_TILES + i) * TB, base + ((int64_t)tl.at(at + i) * a.kv_heads + kvh) * TB, TB, &raw_full[s]);
    };
    // a query's index in the call's queries, or -1 past the run
    auto query = [&](int qi) -> int64_t { return qi < nq ? (int64_t)(run * a.R + qi / G) * a.heads + kvh * G + qi % G : -1; };
    if (warp < 4) {
        // the queries, rows of HD floats far from one another, by bulk copies (none of a padding or refused row)
        const int64_t th = kv4_row_state(base, qpos, a.capacity) ? -1 : query(q0 + threadIdx.x);
        const uint32_t rows = __ballot_sync(0xffffffffu, th >= 0);
        if (lane == 0) mbar_expect_tx(&q_raw, __popc(rows) * HD * 4);
        __syncwarp();
        if (th >= 0) bulk_load(qs + threadIdx.x * pm_q_row(HD), a.q + th * HD, HD * 4, &q_raw);
    } else if (warp == PM_RAW_WARP && lane == 0) {
        for (int j = 0; j < min(steps, 2); ++j) raw_load(j);
    }
    __syncwarp();
    pm_pair_wait<NC>();
    const uint32_t tmem = tmem_base;
    auto live = [&](int it, int r) {        // position r of list item it is seen by some row of the CTA (of the pair)
        return it < i1 && seen(tl.at(it) * KV4_P + r);
    };
    auto raw_step = [&](int j) -> const uint8_t* { return raw + j % PM_RAW * PM_TILES * TB; };

    // Registers: 512 threads of 128 at launch; 168 + 2 * 152 + 40 a thread of the four warpgroups = these 512.
    if (warp < 4) {
        // ---- a query a thread
        regs_inc<168>();
        const uint32_t row = tmem + ((uint32_t)(32 * warp) << 16);
        const int64_t th = query(q0 + threadIdx.x);
        Vis vis{0, 0, 0};
        int state = 1;
        if (th >= 0) {
            state = kv4_row_state(base, qpos, a.capacity);
            if (!state) vis = visible(qpos, a.window, a.sinks);
        }
        float ks;
        {
            // Q's planes: 2^13..2^14 at the row's largest value, dims in the order 0 4 1 5 2 6 3 7
            const float f = a.scale * 1.4426950408889634f;
            const float4* x = reinterpret_cast<const float4*>(qs + threadIdx.x * pm_q_row(HD));
            float mx = 0.f;
            pm_wait(&q_raw, 0u, a.err, abort);
            const bool use = !state;        // (a padding row's query may hold anything: it enters as zeros)
            if (use)
#pragma unroll 8
                for (int i = 0; i < HD / 4; ++i) {
                    const float4 v = x[i];
                    mx = fmaxf(mx, fmaxf(fmaxf(fabsf(v.x * f), fabsf(v.y * f)), fmaxf(fabsf(v.z * f), fabsf(v.w * f))));
                }
            const int e = mx > 0.f && mx <= FLT_MAX ? min(100, 13 - ilogbf(mx)) : 0;      // (-114 at least)
            const float up = ldexpf(1.f, e);
            ks = ldexpf(1.f, -e);
#pragma unroll 1
            for (int i = 0; i < HD / 64; ++i) {
                uint32_t hi[32], lo[32];
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f), w = v;
                    if (use) {
                        v = x[16 * i + 2 * c];
                        w = x[16 * i + 2 * c + 1];
                    }
                    split_h2(f2(v.x * f * up, w.x * f * up), hi[4 * c], lo[4 * c]);
                    split_h2(f2(v.y * f * up, w.y * f * up), hi[4 * c + 1], lo[4 * c + 1]);
                    split_h2(f2(v.z * f * up, w.z * f * up), hi[4 * c + 2], lo[4 * c + 2]);
                    split_h2(f2(v.w * f * up, w.w * f * up), hi[4 * c + 3], lo[4 * c + 3]);
                }
                tmem_st32(row + TM_QH + 32 * i, hi);
                tmem_st32(row + TM_QL + 32 * i, lo);
            }
            tmem_st_wait();
            tc_before();
            __syncwarp();
            if (lane == 0) {
                pm_arrive(&q_read);
                pm_arrive(&q_full);
            }
        }
        // (queries that see nothing, or are none, need no mask: their output is not read)
        const int w_min_n = __reduce_min_sync(0xffffffffu, vis.n > 0 ? vis.n : INT_MAX), w_max_first = __reduce_max_sync(0xffffffffu, vis.first);
        float m = -INFINITY, l = 0.f;
        uint32_t poison = 0u;               // blocks of the output that a seen NaN reached
        for (int j = 0; j < steps; ++j) {
            const uint32_t sbuf = row + TM_S + (j & 1) * 128;
            pm_wait(&s_full[j & 1], (uint32_t)(j / 2 & 1), a.err, abort);
            tc_after();
            const int at = i0 + PM_TILES * j;
            // every query of the warp sees all of column group g (two tiles)
            auto full = [&](int g) {
                const int it = at + 2 * g;
                return it + 1 < i1 && tl.at(it) * KV4_P >= w_max_first && tl.at(it + 1) * KV4_P + KV4_P <= w_min_n;
            };
            // bit n: this query sees column 32 g + n
            auto seen32 = [&](int g) {
                uint32_t b = 0u;
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const int it = at + 2 * g + t;
                    if (it < i1) b |= slots16(seen16(vis, tl.at(it) * KV4_P)) << (4 * t);
                }
                return b;
            };
            // every query of the warp sees all of the step (most steps): a form without masks, so that what most steps run is
            // short (the roles' code outgrows the instruction caches: no instruction was a warp's most frequent wait)
            const bool clear = at + PM_TILES <= i1 && tl.at(at) * KV4_P >= w_max_first && (tl.at(at + PM_TILES - 1) + 1) * KV4_P <= w_min_n;
            auto step = [&](auto masked) {
                constexpr bool MASKED = decltype(masked)::value;
                // a group's scores: those not seen to -inf (the loops are kept rolled: unrolled, the three roles' code outgrew the
                // instruction caches and a step took twice as long; two groups at a time, one's load behind the other's work)
                auto mask = [&](int g, uint32_t (&r)[32]) {
                    if (MASKED && !full(g)) {
                        const uint32_t b = seen32(g);
#pragma unroll
                        for (int i = 0; i < 32; ++i) r[i] = b >> i & 1u ? r[i] : 0xFF800000u;
                    }
                };
                uint32_t ra[32], rb[32];
                float mx = -INFINITY;
#pragma unroll 1
                for (int g = 0; g < 4; g += 2) {
                    tmem_ld32(sbuf + 32 * g, ra);
                    tmem_ld32(sbuf + 32 * g + 32, rb);
                    tmem_ld_wait(ra);
                    tmem_ld_wait(rb);
                    mask(g, ra);
                    mask(g + 1, rb);
#pragma unroll
                    for (int i = 0; i < 32; ++i) mx = fmaxf(mx, fmaxf(__uint_as_float(ra[i]), __uint_as_float(rb[i])));
                }
                tmem_ld32(sbuf, ra);            // the first group again, behind the maximum's work
                const StepCare<NB>& cr = care[j % PM_SLOTS];
                const float kj = cr.big_keys ? 8.f * ks : ks;
                // reference maxima are whole (in log2 units), so that these factors are exact powers of two
                mx = ceilf(mx * kj);
                float f = 1.f;
                if (mx > m + ATT_SLACK) {
                    f = pow2i(m - mx);
                    l *= f;
                    m = mx;
                }
                float mu = mx == -INFINITY ? 0.f : mx - PM_WEIGHT_BITS;
                if (mx - mu > PM_WEIGHT_BITS) mu = mx;          // (a maximum past 2^24: the difference was rounded up)
                const float back = mx == -INFINITY ? 0.f : pow2i(mu - m);
                factor[j % PM_SLOTS][threadIdx.x] = make_float2(f, back);
                if (cr.any_nan) {
                    // a value row with a NaN enters as zeros: it reaches the rows that see it here, and no other
                    for (int g = 0; g < 4; ++g) {
                        const uint32_t see = seen32(g);
                        for (int b = 0; b < NB; ++b)
                            if (cr.nan[b][g] & see) poison |= 1u << b;
                    }
                }
                const uint64_t k2 = f2(kj, kj), m2 = f2(-mu, -mu);
                uint64_t sum = f2(0.f, 0.f);
                // a group's weights in place of its scores: 16 columns of their roundings, 16 of what those left
                auto weights = [&](int g, uint32_t (&r)[32]) {
                    uint32_t lo[16];
                    mask(g, r);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float2 x = unf2(fma2(f2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), k2, m2));
                        const uint64_t p = f2(ex2(x.x), ex2(x.y));
                        sum = add2(sum, p);
                        split_h2(p, r[i], lo[i]);
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) r[16 + i] = lo[i];
                    tmem_st32(sbuf + 32 * g, r);
                };
#pragma unroll 1
                for (int g = 0; g < 4; g += 2) {
                    tmem_ld_wait(ra);
                    tmem_ld32(sbuf + 32 * g + 32, rb);
                    weights(g, ra);
                    tmem_ld_wait(rb);
                    if (g == 0) tmem_ld32(sbuf + 64, ra);
                    weights(g + 1, rb);
                }
                const float2 x = unf2(sum);
                l = __fmaf_rn(x.x + x.y, back, l);
                tmem_st_wait();
            };
            if (clear) step(std::false_type{});
            else step(std::true_type{});
            tc_before();
            __syncwarp();
            if (lane == 0) pm_arrive(&p_full[j & 1]);
        }
        if (state) l = state == 2 ? NAN : 0.f;
        fin_l[threadIdx.x] = l;
        fin_poison[threadIdx.x] = poison;
        if (a.S > 1 && th >= 0) reinterpret_cast<float2*>(a.ml)[th * a.S + sp] = make_float2(state ? -INFINITY : m, l);
        asm volatile("bar.sync 2, 384;" ::: "memory");
    } else if (warp < PM_MMA_WARP) {
        // ---- codes to planes, and the output
        regs_inc<152>();
        const int w = warp - PM_DQ_WARP, g = lane >> 2, c = lane & 3;
        auto all_live = [&](int at) {       // every position of a step's tiles is seen by some row
            return at + PM_TILES <= i1 && tl.at(at) * KV4_P >= seen.first && (tl.at(at + PM_TILES - 1) + 1) * KV4_P <= seen.n;
        };
        auto arrived = [&](int j) {         // step j's raw tiles, and what its values' scales call for
            pm_wait(&raw_full[j % PM_RAW], (uint32_t)(j / PM_RAW & 1), a.err, abort);
            pm_wait(&care_full[j % PM_RAW], (uint32_t)(j / PM_RAW & 1), a.err, abort);
        };
        // K' of step j (a CTA of a pair: its half of the positions): (tile, half) units, a position's 8 dims x NB a lane
        auto keys = [&](int j) {
            uint8_t* kj = kh + j % NP * 2 * PL;
            const __half2 k2 = __float2half2_rn(care[j % PM_SLOTS].big_keys ? 0.125f : 1.f);
            const bool whole = all_live(i0 + PM_TILES * j);
#pragma unroll 1
            for (int u = 0; u < 2 / NC; ++u) {
                const int tile = NC == 1 ? w : 4 * cta + w / 2, h = NC == 1 ? u : w & 1;
                const uint8_t* tp = raw_step(j) + tile * TB;
                uint32_t kw[NB], sw[NB / 2];
                lane_words<HD>(tp, h, lane, kw);
                const uint8_t* sc = tp + 16 * HD + (8 * h + g) * NB * 2;
                if constexpr (NB == 4) {
                    const uint2 x = lds64(sc);
                    sw[0] = x.x;
                    sw[1] = x.y;
                } else {
                    sw[0] = *reinterpret_cast<const uint32_t*>(sc);
                }
                if (!whole && !live(i0 + PM_TILES * j + tile, 8 * h + g)) {
#pragma unroll
                    for (int i = 0; i < NB / 2; ++i) sw[i] = 0u;
                }
                const int n = tile / 2 * 32 - KP * cta + g / 2 * 8 + (2 * (tile & 1) + h) * 2 + (g & 1);
                const int off = n / 8 * 1024 + n % 8 * 128;
#pragma unroll
                for (int i = 0; i < NB; ++i) {
                    // odd g takes the blocks of a pair the other way round: a phase's 8 lanes then write 8 different chunks
                    const bool odd = g & 1;
                    const int b = odd ? i ^ 1 : i;
                    const uint32_t word = odd ? kw[i ^ 1] : kw[i];
                    const uint32_t d16 = __byte_perm(sw[i / 2], 0, (i & 1) != odd ? 0x3232 : 0x1010);
                    const __half2 d = __hmul2(bits_h2(d16), k2);
                    uint32_t r[4], hi[4], lo[4];
                    unpack_signed(word, r);
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const __half2 y = __hmul2(bits_h2(r[x]), d);
                        hi[x] = h2_bits(y);
                        lo[x] = h2_bits(__hfma2(bits_h2(r[x]), d, __hneg2(y)));
                    }
                    const int ch = 4 * b + c;
                    uint8_t* dst = kj + ch / 8 * (KP * 128) + off + ((ch % 8) ^ (n % 8)) * 16;
                    *reinterpret_cast<uint4*>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    *reinterpret_cast<uint4*>(dst + PL) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
            }
        };
        auto keys_done = [&](int j) {
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) pm_arrive(&k_full[j % NP]);
        };
        // V' of step j (a CTA of a pair: its half of the dims): 32 positions (two tiles) and half the blocks, or half of the one
        // block, a warp; a lane 8 positions of 4 dims a block. Made in registers, and put in place.
        constexpr int VB = NB / NC;
        const int grp = w / 2, vb0 = VB > 1 ? (w & 1) * (VB / 2) : 0, vbs = VB > 1 ? VB / 2 : 1;
        auto make_as = [&](auto plain, int j, int vb, uint32_t (&hi)[4][4], uint32_t (&lo)[4][4]) {
            constexpr bool PLAIN = decltype(plain)::value;      // all positions live, no scale that calls for care
            const uint8_t* rs = raw_step(j);
            const StepCare<NB>& cr = care[j % PM_SLOTS];
            const __half2 vs2 = __float2half2_rn(PLAIN ? 256.f : cr.vs());
            const int any_nan = PLAIN ? 0 : cr.any_nan, at = i0 + PM_TILES * j, b = VB * cta + vb;
            uint32_t r[4][4], dv[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint8_t* tp = rs + (2 * grp + k / 2) * TB;
                unpack_signed(*reinterpret_cast<const uint32_t*>(tp + 8 * HD + (((k & 1) * 32 + lane) * NB + b) * 4), r[k]);
                const uint16_t* sc = reinterpret_cast<const uint16_t*>(tp + 17 * HD) + (8 * (k & 1) + 2 * c) * NB + b;
                dv[k] = (uint32_t)sc[0] | (uint32_t)sc[NB] << 16;
                if (!PLAIN) {
                    const int it = at + 2 * grp + k / 2, r0 = 8 * (k & 1) + 2 * c;
                    dv[k] &= (live(it, r0) ? 0xFFFFu : 0u) | (live(it, r0 + 1) ? 0xFFFF0000u : 0u);
                }
                if (any_nan) {              // (a NaN scale, above infinity's bits, enters as zero)
                    if ((dv[k] & 0x7FFFu) > 0x7C00u) dv[k] &= 0xFFFF0000u;
                    if ((dv[k] & 0x7FFF0000u) > 0x7C000000u) dv[k] &= 0xFFFFu;
                }
                dv[k] = h2_bits(__hmul2(bits_h2(dv[k]), vs2));
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                if (VB == 1 && x / 2 != (w & 1)) continue;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const __half2 d = bits_h2(dv[k]), y = __hmul2(bits_h2(r[k][x]), d);
                    hi[x][k] = h2_bits(y);
                    lo[x][k] = h2_bits(__hfma2(bits_h2(r[k][x]), d, __hneg2(y)));
                }
            }
        };
        auto make = [&](int j, int vb, uint32_t (&hi)[4][4], uint32_t (&lo)[4][4]) {
            const StepCare<NB>& cr = care[j % PM_SLOTS];
            if (all_live(i0 + PM_TILES * j) && !cr.vmax && !cr.any_nan) make_as(std::true_type{}, j, vb, hi, lo);
            else make_as(std::false_type{}, j, vb, hi, lo);
        };
        auto put = [&](int j, int vb, const uint32_t (&hi)[4][4], const uint32_t (&lo)[4][4]) {
            if (j == 0) pm_wait(&q_read, 0u, a.err, abort);     // (V' takes the place of the staged queries)
            const int ch = (grp & 1) * 4 + c;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                if (VB == 1 && x / 2 != (w & 1)) continue;
                const int dim = 32 * vb + 4 * g + x;
                uint8_t* dst = vh + j % NP * 2 * PL + grp / 2 * (VD * 128) + dim / 8 * 1024 + dim % 8 * 128 + (ch ^ (dim % 8)) * 16;
                *reinterpret_cast<uint4*>(dst) = make_uint4(hi[x][0], hi[x][1], hi[x][2], hi[x][3]);
                *reinterpret_cast<uint4*>(dst + PL) = make_uint4(lo[x][0], lo[x][1], lo[x][2], lo[x][3]);
            }
        };
        auto values_done = [&](int j) {
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) pm_arrive(&v_full[j % NP]);
        };
        auto raw_done = [&](int j) {
            __syncwarp();
            if (lane == 0) pm_arrive(&raw_empty[j % PM_RAW]);
        };
        // the warp's part of the output: queries 32 (w % 4) + lane, dims HD / 2 * (w / 4) ..
        const int qr = 32 * (w & 3) + lane, d0 = HD / 2 * (w / 4);
        const uint32_t otm = tmem + ((uint32_t)(32 * (w & 3)) << 16) + TM_O + d0;
        uint64_t o[HD / 4];
#pragma unroll
        for (int i = 0; i < HD / 4; ++i) o[i] = f2(0.f, 0.f);
        auto product = [&](int j) {         // step j's product is there
            pm_wait(&pv_done, (uint32_t)(j & 1), a.err, abort);
            tc_after();
        };
        auto collect = [&](int j) {         // and goes into the output
            const StepCare<NB>& cr = care[j % PM_SLOTS];
            const float2 fb = factor[j % PM_SLOTS][qr];
            const float f = fb.x, u = (cr.vmax ? 1.f / cr.vs() : 1.f / 256.f) * fb.y;
            const uint64_t f1 = f2(f, f), u1 = f2(u, u);
            if (__any_sync(0xffffffffu, f != 1.f)) {
#pragma unroll
                for (int i = 0; i < HD / 4; ++i) o[i] = mul2(o[i], f1);
            }
#pragma unroll
            for (int x = 0; x < HD / 64; ++x) {
                uint32_t r[32];
                tmem_ld32(otm + 32 * x, r);
                tmem_ld_wait(r);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    o[16 * x + i] = fma2(f2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), u1, o[16 * x + i]);
            }
            tc_before();
            __syncwarp();
            if (lane == 0) pm_arrive(&o_free);
        };
        if constexpr (NC == 1) {
            uint32_t hi[4][4], lo[4][4];
            if (steps > 0) {
                arrived(0);
                keys(0);
                keys_done(0);
            }
            for (int j = 0; j < steps; ++j) {
                if (j + 1 < steps) {
                    arrived(j + 1);
                    pm_wait(&s_full[j & 1], (uint32_t)(j / 2 & 1), a.err, abort);       // (step j's K' is used)
                    keys(j + 1);
                    keys_done(j + 1);
                }
                if (j > 0) {
                    product(j - 1);
                    collect(j - 1);
                }
#pragma unroll 1
                for (int vb = vb0; vb < vb0 + vbs; ++vb) {
                    make(j, vb, hi, lo);
                    put(j, vb, hi, lo);
                }
                values_done(j);
                raw_done(j);
            }
        } else {
            // two steps of K' and V' each: step j + 1 is made while the product of step j - 1 runs (the fences come after
            // other work: the writes have drained by then), and its V' put in the place of that product's
            uint32_t hi[4][4], lo[4][4];
            for (int j = -1; j < steps; ++j) {
                if (j + 1 < steps) {
                    arrived(j + 1);
                    if (j > 0) pm_wait(&s_full[(j - 1) & 1], (uint32_t)((j - 1) / 2 & 1), a.err, abort);        // (step j - 1's K' is used)
                    keys(j + 1);
                    make(j + 1, vb0, hi, lo);
                    keys_done(j + 1);
                    raw_done(j + 1);
                }
                if (j > 0) product(j - 1);
                if (j + 1 < steps) put(j + 1, vb0, hi, lo);
                if (j > 0) collect(j - 1);
                if (j + 1 < steps) values_done(j + 1);
            }
        }
        if (steps > 0) {
            product(steps - 1);
            collect(steps - 1);
        }
        asm volatile("bar.sync 2, 384;" ::: "memory");
        {
            // the warp's 32 half rows by way of shared memory (a thread's own would go out 16 bytes a line at a time)
            const bool whole = a.S == 1;
            const int r_first = q0 / G;
            const float l = fin_l[qr];
            const float f = l == 0.f ? 0.f : !whole ? 1.f : 1.f / l;    // (a refused row's NaN stays; nothing visible: zeros)
            const uint32_t poison = fin_poison[qr];
            uint8_t* st = os + w * 32 * pm_o_row(HD);
#pragma unroll
            for (int i = 0; i < HD / 4; i += 2) {
                const float g1 = poison >> ((d0 + 2 * i) / 32) & 1u ? NAN : f;
                const float2 x = unf2(o[i]), y = unf2(o[i + 1]);
                *reinterpret_cast<float4*>(st + lane * pm_o_row(HD) + 8 * i) =
                    g1 == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(x.x * g1, x.y * g1, y.x * g1, y.y * g1);
            }
            __syncwarp();
            constexpr int L = HD / 8;           // lanes a half row
            const int qi = q0 + qr, mine = qi < nq ? (qi / G - r_first) * a.heads + qi % G : -1;     // (its row and head from the CTA's first row's)
            const int64_t th0 = (int64_t)(run * a.R + r_first) * a.heads + kvh * G;
            float* dst = (whole ? a.out + th0 * HD : a.part + (th0 * a.S + sp) * HD) + d0 + 4 * (lane % L);
            const int64_t pitch = whole ? HD : (int64_t)a.S * HD;
#pragma unroll
            for (int r = 0; r < 32; r += 32 / L) {
                const int th = __shfl_sync(0xffffffffu, mine, r + lane / L);
                const float4 v = *reinterpret_cast<const float4*>(st + (r + lane / L) * pm_o_row(HD) + 16 * (lane % L));
                if (th >= 0) *reinterpret_cast<float4*>(dst + th * pitch) = v;
            }
        }
    } else {
        regs_dec<40>();
        if (warp == PM_MMA_WARP && cta == 0 && lane == 0 && steps > 0) {
            // ---- one thread (of a pair: for both) issues the MMAs. The products with remainders come first: sums are cut off at their size.
            auto pv = [&](int j) {
                if (j > 0) pm_wait(&o_free, (uint32_t)(j - 1 & 1), a.err, abort);
                pm_wait(&v_full[j % NP], (uint32_t)(j / NP & 1), a.err, abort);
                pm_wait<NC == 2>(&p_full[j & 1], (uint32_t)(j / 2 & 1), a.err, abort);
                if (*abort) return;
                tc_after();
                const uint32_t p = tmem + TM_S + (j & 1) * 128;
                uint64_t v = pm_desc(vh + j % NP * 2 * PL);           // (16-byte units: 2 a step of 16 positions, an atom's HD rows of 128 bytes a step of 64)
#pragma unroll 1
                for (int s = 0; s < PM_P / 64; ++s, v += VD * 8)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const uint32_t ph = p + 64 * s + x / 2 * 32 + x % 2 * 8;
                        pm_mma<NC>(tmem + TM_O, ph, v + 2 * x + (PL >> 4), pm_idesc(HD, NC), s > 0 || x > 0);
                        pm_mma<NC>(tmem + TM_O, ph + 16, v + 2 * x, pm_idesc(HD, NC), 1u);
                    }
                v = pm_desc(vh + j % NP * 2 * PL);
#pragma unroll 1
                for (int s = 0; s < PM_P / 64; ++s, v += VD * 8)
#pragma unroll
                    for (int x = 0; x < 4; ++x) pm_mma<NC>(tmem + TM_O, p + 64 * s + x / 2 * 32 + x % 2 * 8, v + 2 * x, pm_idesc(HD, NC), 1u);
                pm_commit<NC>(&pv_done);
            };
            pm_wait(&q_full, 0u, a.err, abort);
            for (int j = 0; j < steps; ++j) {
                pm_wait<NC == 2>(&k_full[j % NP], (uint32_t)(j / NP & 1), a.err, abort);
                if (j > 1) pm_wait(&pv_done, (uint32_t)(j & 1), a.err, abort);      // the weights that this score buffer held are used
                if (*abort) break;
                tc_after();
                const uint32_t d = tmem + TM_S + (j & 1) * 128;
                uint64_t k = pm_desc(kh + j % NP * 2 * PL);
#pragma unroll 1
                for (int s = 0; s < HD / 64; ++s, k += KP * 8)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        pm_mma<NC>(d, tmem + TM_QH + 32 * s + 8 * x, k + 2 * x + (PL >> 4), pm_idesc(PM_P, NC), s > 0 || x > 0);
                        pm_mma<NC>(d, tmem + TM_QL + 32 * s + 8 * x, k + 2 * x, pm_idesc(PM_P, NC), 1u);
                    }
                k = pm_desc(kh + j % NP * 2 * PL);
#pragma unroll 1
                for (int s = 0; s < HD / 64; ++s, k += KP * 8)
#pragma unroll
                    for (int x = 0; x < 4; ++x) pm_mma<NC>(d, tmem + TM_QH + 32 * s + 8 * x, k + 2 * x, pm_idesc(PM_P, NC), 1u);
                pm_commit<NC>(&s_full[j & 1]);
                if (j > 0) pv(j - 1);
            }
            pv(steps - 1);
            if (*abort) {
                pm_commit<NC>(&drained);
                mbar_drain(&drained, 0u);
            }
        } else if (NC == 2 && warp == PM_MMA_WARP && lane == 0 && steps > 0) {
            // ---- a pair's other CTA: what the MMAs wait for, on to the first CTA in the order of its waits, one arrival for all
            // that a product waits for (made by the warps themselves, each across the pair, they cost them 400 cycles a time)
            auto wait = [&](uint64_t* bar, int n) { pm_wait(bar, (uint32_t)(n & 1), a.err, abort); };
            auto forward = [&](uint64_t* bar) {
                tc_after();
                tc_before();
                pm_arrive_lead(bar);
            };
            auto pv = [&](int j) {
                if (j > 0) wait(&o_free, j - 1);
                wait(&v_full[j % NP], j / NP);
                wait(&p_full[j & 1], j / 2);
                forward(&p_full[j & 1]);
            };
            wait(&q_full, 0);
            for (int j = 0; j < steps; ++j) {
                wait(&k_full[j % NP], j / NP);
                forward(&k_full[j % NP]);
                if (j > 0) pv(j - 1);
            }
            pv(steps - 1);
        } else if (warp == PM_RAW_WARP && lane == 0) {
            // ---- raw tiles
            int issued = min(steps, 2);
            for (int j = 2; j < steps; ++j) {
                // (the places of steps 2 and 3 held the staged queries)
                if (j >= PM_RAW) pm_wait(&raw_empty[j % PM_RAW], (uint32_t)((j / PM_RAW + 1) & 1), a.err, abort);
                else if (j == 2) pm_wait(&q_read, 0u, a.err, abort);
                if (*abort) break;
                fence_proxy_async();
                raw_load(j);
                issued = j + 1;
            }
            if (*abort) {
                mbar_drain(&q_raw, 0u);
                for (int j = max(0, issued - PM_RAW); j < issued; ++j) mbar_drain(&raw_full[j % PM_RAW], (uint32_t)(j / PM_RAW & 1));
            }
        } else if (warp == PM_CARE_WARP) {
            // ---- what the scales of a step call for: nothing, unless a value's is 2 or more, a key's 2^13 or more, or one NaN (or
            // what lies in unseen places looks so). A slot's step of PM_SLOTS before is behind every warp: its raw tiles' place
            // was given up twice.
            constexpr int words = KV4_P * NB / 2;           // of two fp16 scales, of a tile
            uint32_t used = 0u;                             // slots that are not clear
            for (int j = 0; j < steps; ++j) {
                const int at = i0 + PM_TILES * j, slot = j % PM_SLOTS;
                pm_wait(&raw_full[j % PM_RAW], (uint32_t)(j / PM_RAW & 1), a.err, abort);
                uint32_t any = 0u;
                for (int t = 0; t < PM_TILES; ++t)
                    if (lane < words && at + t < i1) {
                        const uint32_t k = reinterpret_cast<const uint32_t*>(raw_step(j) + t * TB + 16 * HD)[lane];
                        any |= reinterpret_cast<const uint32_t*>(raw_step(j) + t * TB + 17 * HD)[lane];
                        any |= k & k << 1 & k << 2;             // (the exponent's top three bits: 2^13, infinity or NaN)
                    }
                if (__any_sync(0xffffffffu, any & 0x40004000u) || (used >> slot & 1u)) {
                    StepCare<NB>& cr = care[slot];
                    if (lane == 0) cr.clear();
                    __syncwarp();
                    uint32_t big = 0u;
                    bool nans = false, big_keys = false;
                    for (int t = 0; t < PM_TILES; ++t) {
                        if (lane >= words || at + t >= i1) continue;
                        const uint32_t x = reinterpret_cast<const uint32_t*>(raw_step(j) + t * TB + 17 * HD)[lane];
                        const uint32_t k = reinterpret_cast<const uint32_t*>(raw_step(j) + t * TB + 16 * HD)[lane];
                        for (int e = 0; e < 2; ++e) {
                            const int r = (2 * lane + e) / NB, b = (2 * lane + e) % NB;
                            const uint32_t d = (x >> (16 * e)) & 0x7FFFu, kd = (k >> (16 * e)) & 0x7FFFu;
                            if (!live(at + t, r)) continue;
                            big_keys |= kd >= 0x7000u && kd <= 0x7C00u;
                            if (d < 0x4000u) continue;
                            if (d > 0x7C00u) {
                                nans = true;
                                atomicOr(&cr.nan[b][t / 2], 1u << (8 * (r % 8 / 2) + 2 * (2 * (t & 1) + r / 8) + r % 2));
                            } else {
                                big = max(big, __float_as_uint(__half2float(__ushort_as_half((unsigned short)d))));
                            }
                        }
                    }
                    big = __reduce_max_sync(0xffffffffu, big);
                    nans = __any_sync(0xffffffffu, nans);
                    big_keys = __any_sync(0xffffffffu, big_keys);
                    if (lane == 0) {
                        cr.vmax = big;
                        cr.any_nan = nans;
                        cr.big_keys = big_keys;
                    }
                    used = big || nans || big_keys ? used | 1u << slot : used & ~(1u << slot);
                }
                __syncwarp();
                if (lane == 0) pm_arrive(&care_full[j % PM_RAW]);
            }
        }
    }
    tc_before();
    __syncwarp();
    pm_pair_arrive<NC>();
    pm_pair_wait<NC>();                     // (nothing arrives at a pair's other CTA, and no MMA uses it, after this)
    __syncthreads();
    if (warp == 0) {
        tc_after();
        if constexpr (NC == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
    if (a.S == 1 || q0 >= nq) return;
    // (128 registers for all again: the join compiled for the fewest kept its partials in local memory)
    if (warp < PM_MMA_WARP) regs_dec<128>();
    else regs_inc<128>();
    if (!last_ticket(a.tickets + ((int64_t)run * a.kv_heads + kvh) * q_blocks + qb, a.S)) return;
    join_ranges<HD, PM_THREADS>(a.ml, a.part, a.out, a.S, min(PM_Q, nq - q0), a.S, reinterpret_cast<float*>(smem),
                                RowMap{(int64_t)run * a.R * a.heads + kvh * G, q0, G, a.heads});
}

template <int HD, int NC> void launch_mma(const Kv4Att& a, int q_blocks, cudaStream_t s)
{
    auto kern = k_kv4_attn_mma<HD, NC>;
    constexpr int smem = pm_smem(HD, NC);
    static std::atomic<bool> done[64];
    ensure_smem_attr(kern, smem, done);
    // (launched plainly: it takes all of an SM's tensor memory, so it does not start beside another kernel's end)
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(q_blocks * a.S, a.kv_heads, a.T / a.R);
    cfg.blockDim = dim3(PM_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = NC;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    WL_CUDA(cudaLaunchKernelEx(&cfg, kern, a, q_blocks));
    note_launch();
}

}  // namespace

void kv4_attention_mma(const Kv4Att& a, int head_dim, int q_blocks, bool pairs, cudaStream_t s)
{
    if (head_dim == 64) pairs ? launch_mma<64, 2>(a, q_blocks, s) : launch_mma<64, 1>(a, q_blocks, s);
    else pairs ? launch_mma<128, 2>(a, q_blocks, s) : launch_mma<128, 1>(a, q_blocks, s);
}

}  // namespace k
}  // namespace wl
