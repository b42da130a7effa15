// Sampling of many rows in one launch: temperature, top-k, top-p and min-p, each row with its own options and its own
// uniform draw.
//
//   temperature <= 0: the greedy id (wl_argmax's rule).
//   p[i] = exp((x[i] - max) / temperature) in double, the difference in float (Sampler.Sample's arithmetic); NaN and -inf logits have none, and every id at the maximum has 1.
//   The ids in order: logit descending, equal logits by ascending id. Kept is a prefix of that order: the top_k first ids
//   (top_k > 0), of these the shortest prefix whose sum reaches top_p * (their sum) (top_p < 1), of these the ones with
//   p >= min_p (min_p > 0), and at least the first. The choice is the first id at which the running sum reaches draw * (the
//   sum of what is kept). With no filter the running sum goes in id order, as Sampler.Sample's does at top_p >= 1
//   (src/Engine.cs:361-380).
//
// A cluster of CTAs takes a row; each keeps its slice of the logits in shared memory, so the row is read once. Nothing is
// sorted: each of the three cuts (the k-th id, the nucleus's end, the pick) is a selection in that order. A histogram over
// the logits (2048 bins of equal width from the maximum down; one rounded product, so the bins keep the order) gives the
// bin that the cut falls in, its few ids are gathered to one CTA and ranked by counting, each against each. A bin of more
// than SR_CAP ids (ties, or a row whose values are far from evenly spread) is cut again by the bits of the logits and then
// by ids. The probabilities are summed as 64-bit integers, multiples of 2^-F with F = 62 - ceil(log2 V) (44 for
// 151936 ids), 51 at most, so that every sum is exact and does not depend on the order of the atomics; rounding them moves a
// boundary between two ids by at most V * 2^-(F+1), 4e-9 of the sum at 151936 ids, and as a rule by the square root of V such
// halves, 1e-11.
//
// Measured: 12.1 us for a row of 32000 logits with a top-k, 24.7 us for 8 rows of 151936 with mixed filters, 77.7 us for 64 rows
// of 128256 (33 MB: 0.42 TB/s). The time follows the rows: other draws of the same 8 rows took 26 to 70 us (a row whose nucleus
// ends in a bin of more than SR_CAP ids is cut again), of the 64 rows 57 to 82, each the same to 1 % when repeated. A latency chain, not bandwidth: of a CTA's 45000 cycles with a nucleus 5000 are the load, 17000 the
// histogram of masses (an exponential in double and one or two shared atomics a logit; two CTAs share an SM), 6000 a
// join of the cluster's histograms, 8000 the gather and 7000 the ranking. Two CTAs an SM, 512 threads each: the 512 CTAs of
// 64 rows are 1.7 waves. Tried and slower: every CTA's gathered ids in a list of its own with the counts exchanged (no
// atomics across the cluster: 12.9 / 26.1 / 79.3 us), a table of 256 for the exponential in place of 64.
#include <algorithm>
#include <cfloat>
#include <climits>
#include <cstdint>
#include "wl_common.h"
#include "wl_kernels.h"
#include "wl_launch.cuh"

namespace wl {
namespace k {

namespace {

constexpr int SR_THREADS = 512, SR_WARPS = SR_THREADS / 32;
constexpr int SR_BINS = 2048;               // most histogram bins: 512 a CTA of the cluster, one a thread
constexpr int SR_CAP = SR_THREADS;          // ids ranked at once, one a thread
constexpr int SR_MAX_CLUSTER = 8;
constexpr int SR_SLICE_MAX = 44 * 1024;     // logits a CTA keeps in shared memory; longer slices are read from L2

typedef unsigned long long u64;

__device__ __forceinline__ uint32_t cluster_rank()
{
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// The address of `p` (shared memory of this CTA) in CTA `rank` of the cluster.
template <typename T> __device__ __forceinline__ T* remote(T* p, int rank)
{
    uint64_t a;
    asm("mapa.u64 %0, %1, %2;" : "=l"(a) : "l"((uint64_t)p), "r"(rank));
    return reinterpret_cast<T*>(a);
}

// Floats in an order that integers have: larger value, larger key; -0 as +0.
__device__ __forceinline__ uint32_t order_key(float x)
{
    uint32_t b = __float_as_uint(x);
    if (b == 0x80000000u) b = 0u;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct Item {               // a selected id: its key, id, and the sum up to and with it
    uint32_t key, id;
    u64 cum;
};

// What a row's loops need of it, in registers while they run.
struct RowConst {
    float xmax, inv_w, last_bin;            // the histogram: bin = (xmax / 2 - x / 2) * inv_w
    int frac;
    double inv_t, unit;                     // log2(e) / temperature, 2^F
    int has_k;                              // a top-k cut: ids up to (k_key, k_id) in the order
    uint32_t k_key, k_id;

    __device__ __forceinline__ bool kept(uint32_t key, uint32_t id) const { return !has_k || key > k_key || (key == k_key && id <= k_id); }
    __device__ __forceinline__ int bin0(float x) const
    {
        return (int)fminf((xmax * 0.5f - x * 0.5f) * inv_w, last_bin);      // (NaN, of infinities: the last bin)
    }
    // p 2^F, rounded (below 2^52: adding 2^52 leaves the integer in the sum's low bits)
    __device__ __forceinline__ u64 mass(double p) const
    {
        return (u64)__double_as_longlong(fma(p, unit, 4503599627370496.0)) & 0xFFFFFFFFFFFFFull;
    }
    // exp((x - xmax) / T), 0 for a NaN or -inf x: 2^y by table and polynomial (Tang's table-driven scheme: y = n + j/64 + r,
    // 2^(j/64) from the table, e^(r ln 2) to the fifth power, its remainder below 2^-54). No branch, so that several run
    // side by side.
    __device__ __forceinline__ double prob(float x, const double* exp2_table) const
    {
        const double y = (double)__fsub_rn(x, xmax) * inv_t;
        const bool some = y > -(double)(frac + 2);
        // y 64 to the nearest integer: the low bits of a sum with 1.5 2^52
        const double yy = some ? y : 0.0, z = fma(yy, 64.0, 6755399441055744.0);
        const int i = __double2loint(z);
        const double t = fma(z - 6755399441055744.0, -0.015625, yy) * 0.6931471805599453, t2 = t * t;
        const double e = fma(t2, fma(t2, fma(t, 1.0 / 120, 1.0 / 24), fma(t, 1.0 / 6, 0.5)), 1.0 + t);
        const double m = exp2_table[i & 63] * e;
        const double p = __hiloint2double(__double2hiint(m) + ((i >> 6) << 20), __double2loint(m));
        return x == xmax ? 1.0 : some ? p : 0.0;    // (some is false for a NaN and for -inf)
    }
};

// A row's state in a CTA's shared memory (all of its scalars the same for all threads).
struct Row {
    uint32_t lo[SR_BINS], hi[SR_BINS];      // per bin: a count (lo), or a 64-bit sum in two words
    double exp2_table[64];
    u64 scan[SR_WARPS];
    const float* xs;                        // this CTA's slice
    int n, id0, C, rank, bins;              // its length and first id; the cluster; bins in use
    RowConst c;
    // published by every CTA of the cluster into each
    u64 part[SR_MAX_CLUSTER], best[SR_MAX_CLUSTER], min_part[SR_MAX_CLUSTER];
    uint32_t low[SR_MAX_CLUSTER];
    struct Cut {                            // a crossing bin, the sum before it and in it
        int bin, bin_hi;
        u64 before, sum;
    } cut[2];
    Item item;
    u64 found[2];
    // in CTA 0: the gathered ids, and the range of keys and ids of a crowded bin
    int n_cand;
    uint32_t kmin, kmax, imin, imax;
    uint32_t ckey[SR_CAP], cid[SR_CAP];
    u64 cval[SR_CAP];
    int cbin[SR_CAP];

    __device__ __forceinline__ void add(int b, u64 v, bool count)
    {
        if (count) {
            atomicAdd(&lo[b], 1u);
        } else {
            // a 64-bit sum of two 32-bit words: the add that wraps the low word carries into the high one
            const uint32_t l = (uint32_t)v, old = atomicAdd(&lo[b], l);
            const uint32_t h = (uint32_t)(v >> 32) + (old + l < old ? 1u : 0u);
            if (h) atomicAdd(&hi[b], h);
        }
    }
    // (one thread)
    template <typename T> __device__ __forceinline__ void publish(T* p, T v)
    {
        for (int r = 0; r < C; ++r) *remote(p, r) = v;
    }
};

__device__ __forceinline__ float key_value(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key); }
__device__ __forceinline__ bool valid(float x) { return x > -INFINITY; }

// Sum over the threads before this one, and over all.
__device__ __noinline__ u64 block_before(Row& s, u64 v, u64* total)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    u64 inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
    }
    __syncthreads();
    if (lane == 31) s.scan[warp] = inc;
    __syncthreads();
    u64 b = 0, all = 0;
#pragma unroll
    for (int w = 0; w < SR_WARPS; ++w) {
        const u64 x = s.scan[w];
        if (w < warp) b += x;
        all += x;
    }
    *total = all;
    return b + inc - v;
}

__device__ __forceinline__ void clear_hist(Row& s)
{
    for (int b = threadIdx.x; b < s.bins; b += SR_THREADS) s.lo[b] = s.hi[b] = 0u;
    __syncthreads();
}

// The cluster's histogram joined: this thread's bin (its CTA's share of bins, one a thread), the sum before it, and all.
struct Joined {
    u64 v, before, total;
};
__device__ __noinline__ Joined join(Row& s, bool count)
{
    cluster_sync();                         // every CTA's histogram is complete
    const int share = s.bins / s.C, at = s.rank * share + threadIdx.x, C = s.C;
    Joined j;
    j.v = 0;
    if ((int)threadIdx.x < share) {
        uint32_t l[SR_MAX_CLUSTER], h[SR_MAX_CLUSTER];      // (all CTAs' loads in flight together)
#pragma unroll
        for (int r = 0; r < SR_MAX_CLUSTER; ++r) {
            l[r] = r < C ? *remote(&s.lo[at], r) : 0u;
            h[r] = r < C && !count ? *remote(&s.hi[at], r) : 0u;
        }
#pragma unroll
        for (int r = 0; r < SR_MAX_CLUSTER; ++r) j.v += (u64)l[r] + ((u64)h[r] << 32);
    }
    u64 mine;
    j.before = block_before(s, j.v, &mine);
    if ((int)threadIdx.x < C) *remote(&s.part[s.rank], threadIdx.x) = mine;
    cluster_sync();
    j.total = 0;
#pragma unroll
    for (int r = 0; r < SR_MAX_CLUSTER; ++r) {
        const u64 x = r < C ? s.part[r] : 0ull;
        if (r < s.rank) j.before += x;
        j.total += x;
    }
    return j;
}

// The bin in which base + the running sum first reaches target (1 <= target - base <= total), in s.cut[which] of every CTA;
// clears the list of the gather that follows.
__device__ __forceinline__ void find(Row& s, const Joined& j, u64 target, u64 base, int which = 0)
{
    // (the lanes of the warp that has it write one CTA each)
    const u64 b = base + j.before, e = b + j.v;
    const uint32_t who = __ballot_sync(0xffffffffu, b < target && e >= target);
    if (who) {
        const int src = __ffs(who) - 1, lane = threadIdx.x & 31;
        const u64 cb = __shfl_sync(0xffffffffu, b, src), cv = __shfl_sync(0xffffffffu, j.v, src);
        if (lane < s.C) {
            Row::Cut* cut = remote(&s.cut[which], lane);
            cut->bin = s.rank * (s.bins / s.C) + (int)threadIdx.x - lane + src;
            cut->before = cb;
            cut->sum = cv;
        }
    }
    if (s.rank == 0 && threadIdx.x == 0) {
        s.n_cand = 0;
        s.kmin = s.imin = UINT_MAX;
        s.kmax = s.imax = 0u;
    }
    cluster_sync();
}

// f(i, x) for this CTA's logits, four (i .. i + 3, -inf past the end) at a time.
template <typename F> __device__ __forceinline__ void each_four(const Row& s, const F& f)
{
    const float* xs = s.xs;
    const int n = s.n;
    const bool aligned = ((uintptr_t)xs & 15) == 0;
    for (int i = 4 * threadIdx.x; i < n; i += 4 * SR_THREADS) {
        float x[4];
        if (aligned && i + 4 <= n) {
            *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(xs + i);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = i + k < n ? xs[i + k] : -INFINITY;
        }
        f(i, x);
    }
}

// f(key, id, mass or 1) for this CTA's ids whose logit pre takes, that in(key, id) takes, that the top-k cut keeps and that
// have a mass.
template <typename Pre, typename In, typename F>
__device__ __forceinline__ void each(const Row& s, const RowConst& c, bool count, const Pre& pre, const In& in, const F& f)
{
    const int id0 = s.id0;
    each_four(s, [&](int i, const float (&x)[4]) {
        bool take[4], any = false;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            take[k] = pre(x[k]) && valid(x[k]);
            any |= take[k];
        }
        if (!any) return;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t key = order_key(x[k]), id = (uint32_t)(id0 + i + k);
            if (!take[k] || !in(key, id) || !c.kept(key, id)) continue;
            const u64 m = count ? 1ull : c.mass(c.prob(x[k], s.exp2_table));
            if (m) f(key, id, m);
        }
    });
}

// Those ids to CTA 0's list (up to SR_CAP of them; s.n_cand there counts all).
template <typename Pre, typename In> __device__ __forceinline__ void gather(Row& s, const RowConst& c, bool count, const Pre& pre, const In& in)
{
    Row* lead = remote(&s, 0);
    each(s, c, count, pre, in, [&](uint32_t key, uint32_t id, u64 m) {
        // one add for the lanes that are here together
        const uint32_t here = __activemask(), lane = threadIdx.x & 31;
        int at = 0;
        if (lane == __ffs(here) - 1) at = atomicAdd(&lead->n_cand, __popc(here));
        at = __shfl_sync(here, at, __ffs(here) - 1) + __popc(here & ((1u << lane) - 1u));
        if (at < SR_CAP) {
            lead->ckey[at] = key;
            lead->cid[at] = id;
            lead->cval[at] = m;
        }
    });
    cluster_sync();
}

// The item at which the running sum (of ones, or of masses) reaches target; the level-0 histogram is joined in j.
__device__ __noinline__ Item select(Row& s, const Joined j0, u64 target, bool count)
{
    find(s, j0, target, 0);
    const RowConst c = s.c;
    const int bin = s.cut[0].bin;
    u64 before = s.cut[0].before;
    bool deep = false;                      // past level 0: the ids with keys [klo, khi] and ids [ilo, ihi]
    uint32_t klo = 0u, khi = UINT_MAX, ilo = 0u, ihi = UINT_MAX;
    Row* lead = remote(&s, 0);
    auto pre = [&](float x) { return deep || c.bin0(x) == bin; };
    auto in = [&](uint32_t key, uint32_t id) { return key >= klo && key <= khi && id >= ilo && id <= ihi; };
    // (a cut by keys leaves 2^-9 of their range at most, one by ids of theirs: at most nine rounds)
#pragma unroll 1
    for (int round = 0; round < 16; ++round) {
        gather(s, c, count, pre, in);
        const int nc = lead->n_cand;
        if (nc <= SR_CAP) {
            if (s.rank == 0 && (int)threadIdx.x < nc) {
                const uint32_t key = s.ckey[threadIdx.x], id = s.cid[threadIdx.x];
                u64 cum = before;
                for (int q = 0; q < nc; ++q)
                    if (s.ckey[q] > key || (s.ckey[q] == key && s.cid[q] <= id)) cum += s.cval[q];
                if (cum >= target && cum - s.cval[threadIdx.x] < target) s.publish(&s.item, Item{key, id, cum});
            }
            cluster_sync();
            return s.item;
        }
        // a crowded range: cut it by the bits of its keys, or, all keys equal, by ids
        uint32_t k0 = UINT_MAX, k1 = 0u, d0 = UINT_MAX, d1 = 0u;
        each(s, c, count, pre, in, [&](uint32_t key, uint32_t id, u64) {
            k0 = min(k0, key);
            k1 = max(k1, key);
            d0 = min(d0, id);
            d1 = max(d1, id);
        });
        k0 = __reduce_min_sync(0xffffffffu, k0);
        k1 = __reduce_max_sync(0xffffffffu, k1);
        d0 = __reduce_min_sync(0xffffffffu, d0);
        d1 = __reduce_max_sync(0xffffffffu, d1);
        if ((threadIdx.x & 31) == 0 && k0 <= k1) {
            atomicMin(&lead->kmin, k0);
            atomicMax(&lead->kmax, k1);
            atomicMin(&lead->imin, d0);
            atomicMax(&lead->imax, d1);
        }
        cluster_sync();
        klo = lead->kmin; khi = lead->kmax; ilo = lead->imin; ihi = lead->imax;
        deep = true;
        const bool by_id = klo == khi;
        const uint32_t width = by_id ? ihi - ilo : khi - klo;
        const int shift = max(0, 32 - __clz(width) - (31 - __clz(s.bins)));
        clear_hist(s);
        each(s, c, count, pre, in, [&](uint32_t key, uint32_t id, u64 m) { s.add((by_id ? id - ilo : khi - key) >> shift, m, count); });
        const Joined j = join(s, count);
        find(s, j, target, before);
        before = s.cut[0].before;
        const uint32_t from = (uint32_t)s.cut[0].bin << shift, upto = from + ((1u << shift) - 1u);
        if (by_id) {
            const uint32_t i0 = ilo;
            ilo = i0 + from;
            ihi = min(ihi, i0 + upto);
        } else {
            const uint32_t top = khi;
            khi = top - from;
            klo = top - klo > upto ? top - upto : klo;
        }
    }
    return s.item;
}

__device__ __forceinline__ u64 share_of(double part, u64 sum)      // the sum that the running sum has to reach: 1 .. sum
{
    const double t = ceil(part * (double)sum);
    return min(sum, t > 1.0 ? (u64)t : 1ull);
}

// f(i, q) for every pair of list items i < n and q < n, the q's of an i shared by a group of g lanes (whose lane 0 gets true
// from owner()): g so that the pairs spread over the CTA.
struct Pairs {
    int i, sub, g;
    __device__ __forceinline__ explicit Pairs(int n)
    {
        g = n <= 16 ? 32 : n <= 32 ? 16 : n <= 64 ? 8 : n <= 128 ? 4 : n <= 256 ? 2 : 1;
        i = threadIdx.x / g;
        sub = threadIdx.x & (g - 1);
    }
    template <typename T> __device__ __forceinline__ T sum(T v) const
    {
        for (int o = 1; o < g; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    }
};

// CTA 0's list of n ids (0 < n <= SR_CAP), among them the first k of the order: its top-k, top-p, min-p and pick.
__device__ __noinline__ void finish_list(Row& s, int n, int k, const wl_sample_opts& o, int32_t* out)
{
    const int tid = threadIdx.x;
    const RowConst c = s.c;
    const Pairs pr(n);
    uint32_t key = 0, id = 0;
    int rank = 0;
    if (pr.i < n) {
        key = s.ckey[pr.i];
        id = s.cid[pr.i];
        for (int q = pr.sub; q < n; q += pr.g) rank += s.ckey[q] > key || (s.ckey[q] == key && s.cid[q] < id);
    }
    rank = pr.sum(rank);
    __syncthreads();
    if (pr.i < n && pr.sub == 0) {
        s.ckey[rank] = key;
        s.cid[rank] = id;
    }
    __syncthreads();
    k = min(k, n);
    double p = 0.0;
    u64 m = 0, all;
    if (tid < k) {
        p = c.prob(key_value(s.ckey[tid]), s.exp2_table);
        m = c.mass(p);
    }
    const u64 cum = block_before(s, m, &all) + m;
    u64 sum = all;
    if (o.top_p < 1.0) {
        const u64 t = share_of(o.top_p, sum);
        if (cum >= t && cum - m < t) s.found[0] = cum;      // (one thread: m > 0)
        __syncthreads();
        sum = s.found[0];
    }
    if (o.min_p > 0.0) {
        const int above = __syncthreads_count(tid < k && p >= o.min_p);
        if (tid == above - 1) s.found[1] = cum;
        __syncthreads();
        sum = max(1ull, min(sum, above ? s.found[1] : 0ull));
    }
    const u64 t = share_of(o.draw, sum);
    if (cum >= t && cum - m < t) *out = (int32_t)s.cid[tid];
}

// CTA 0's list of n ids with their masses: those of the bin that the nucleus ends in (nb, the sum before it nbefore; nb < 0:
// no nucleus, the kept sum is `sum`), and of the bins p_lo .. p_hi that the pick falls in whichever id that is (pbefore: the
// sum before p_lo). over: the sum of the ids with p >= min_p.
__device__ __noinline__ void finish_bins(Row& s, int n, int nb, u64 nbefore, u64 ntarget, int p_lo, int p_hi, u64 pbefore, u64 sum, u64 over,
                                         double draw, int32_t* out)
{
    const RowConst c = s.c;
    for (int i = threadIdx.x; i < n; i += SR_THREADS) s.cbin[i] = c.bin0(key_value(s.ckey[i]));
    __syncthreads();
    const Pairs pr(n);
    uint32_t key = 0, id = 0;
    int bin = -1;
    u64 m = 0, cn = 0, cp = 0;
    if (pr.i < n) {
        key = s.ckey[pr.i];
        id = s.cid[pr.i];
        m = s.cval[pr.i];
        bin = s.cbin[pr.i];
        for (int q = pr.sub; q < n; q += pr.g) {
            const uint32_t k = s.ckey[q];
            if (k > key || (k == key && s.cid[q] <= id)) {
                const int b = s.cbin[q];
                const u64 v = s.cval[q];
                cn += b == nb ? v : 0ull;
                cp += b >= p_lo && b <= p_hi ? v : 0ull;
            }
        }
    }
    cn = nbefore + pr.sum(cn);
    cp = pbefore + pr.sum(cp);
    if (nb >= 0) {
        if (bin == nb && cn >= ntarget && cn - m < ntarget) s.found[0] = cn;
        __syncthreads();
        sum = s.found[0];
    }
    sum = max(1ull, min(sum, over));
    const u64 t = share_of(draw, sum);
    if (bin >= p_lo && bin <= p_hi && cp >= t && cp - m < t) *out = (int32_t)id;
}

__global__ void __launch_bounds__(SR_THREADS, 2) k_sample_rows(const float* logits, int64_t ld, int V, int frac,
                                                               const wl_sample_opts* opts, int32_t* ids, int slice, int in_smem)
{
    extern __shared__ __align__(16) uint8_t smem[];
    Row& s = *reinterpret_cast<Row*>(smem);
    pdl_trigger();
    pdl_wait();
    const int row = blockIdx.y, C = gridDim.x, rank = (int)cluster_rank(), tid = threadIdx.x;
    const float* x = logits + (int64_t)row * ld;
    const wl_sample_opts o = opts[row];
    const int id0 = rank * slice, n = max(0, min(slice, V - id0));
    const bool greedy = !(o.temperature > 0.0);
    cluster_arrive();                       // (waited for before another CTA's memory is written)
    if (tid < 64) s.exp2_table[tid] = exp2(tid * 0.015625);
    // the slice, and its largest value (lowest id) and smallest value above -inf
    float* keep = in_smem ? reinterpret_cast<float*>(smem + (sizeof(Row) + 15) / 16 * 16) : nullptr;
    u64 best = 0;
    uint32_t low = UINT_MAX;
    {
        const float* xs = x + id0;
        float top = -INFINITY, bottom = INFINITY;
        int top_i = -1;
        auto take = [&](int i, float v) {   // (a thread's i ascend: the first of equal values stays)
            if (v > top) {
                top = v;
                top_i = i;
            }
            if (v > -INFINITY) bottom = fminf(bottom, v);
        };
        int done = 0;
        if (((uintptr_t)xs & 15) == 0) {
            const int n4 = n / 4;
            int i = tid;
            for (; i + 3 * SR_THREADS < n4; i += 4 * SR_THREADS) {
                float4 v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = reinterpret_cast<const float4*>(xs)[i + k * SR_THREADS];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int at = i + k * SR_THREADS;
                    if (keep) reinterpret_cast<float4*>(keep)[at] = v[k];
                    take(4 * at, v[k].x);
                    take(4 * at + 1, v[k].y);
                    take(4 * at + 2, v[k].z);
                    take(4 * at + 3, v[k].w);
                }
            }
            for (; i < n4; i += SR_THREADS) {
                const float4 v = reinterpret_cast<const float4*>(xs)[i];
                if (keep) reinterpret_cast<float4*>(keep)[i] = v;
                take(4 * i, v.x);
                take(4 * i + 1, v.y);
                take(4 * i + 2, v.z);
                take(4 * i + 3, v.w);
            }
            done = 4 * n4;
        }
        for (int i = done + tid; i < n; i += SR_THREADS) {
            const float v = xs[i];
            if (keep) keep[i] = v;
            take(i, v);
        }
        if (top_i >= 0) {
            best = (u64)order_key(top) << 32 | (uint32_t)~(uint32_t)(id0 + top_i);
            low = order_key(bottom);
        }
        if (tid == 0) {
            s.xs = keep ? keep : xs;
            s.n = n;
            s.id0 = id0;
            s.C = C;
            s.rank = rank;
            s.bins = min(SR_BINS, 512 * C);
            s.c.frac = frac;
            s.c.last_bin = (float)(s.bins - 1);
            s.c.has_k = 0;
        }
    }
    auto reduce = [&] {
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            const u64 b = __shfl_xor_sync(0xffffffffu, best, d);
            best = b > best ? b : best;
        }
        low = __reduce_min_sync(0xffffffffu, low);
    };
    reduce();
    if ((tid & 31) == 0) {
        s.scan[tid >> 5] = best;
        s.cid[tid >> 5] = low;
    }
    __syncthreads();
    cluster_wait();                         // (every CTA of the cluster has started: its memory may be written)
    if (tid < 32) {
        best = tid < SR_WARPS ? s.scan[tid] : 0;
        low = tid < SR_WARPS ? s.cid[tid] : UINT_MAX;
        reduce();
        if (tid < C) {
            *remote(&s.best[rank], tid) = best;
            *remote(&s.low[rank], tid) = low;
        }
    }
    cluster_sync();
    best = 0;
    low = UINT_MAX;
    for (int r = 0; r < C; ++r) {
        best = s.best[r] > best ? s.best[r] : best;
        low = min(low, s.low[r]);
    }
    const bool lead = rank == 0 && tid == 0;
    // nothing above -inf, or the greedy id. All CTAs take the same branch; nothing of another CTA is read after it.
    if (best == 0 || greedy || !(o.draw >= 0.0 && o.draw < 1.0)) {
        if (lead) ids[row] = !greedy && !(o.draw >= 0.0 && o.draw < 1.0) ? -1 : best == 0 || (greedy && isnan(x[0])) ? 0 : (int32_t)~(uint32_t)best;
        return;
    }
    const bool with_k = o.top_k > 0 && o.top_k < V, sorted = with_k || o.top_p < 1.0 || o.min_p > 0.0;
    const float xmax = key_value((uint32_t)(best >> 32));
    // the histogram's range: down to the smallest value, in halves so that no difference overflows
    const float half_range = xmax * 0.5f - key_value(low) * 0.5f;
    auto width = [&](float range) { return range > 0.f && range <= FLT_MAX ? (float)s.bins / range : 0.f; };
    if (tid == 0) {
        s.c.xmax = xmax;
        s.c.inv_t = 1.4426950408889634 / o.temperature;
        s.c.unit = ldexp(1.0, frac);
        s.c.inv_w = width(half_range);
    }
    Joined j;
    if (with_k) {
        clear_hist(s);
        const RowConst c = s.c;
        each_four(s, [&](int, const float (&v)[4]) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int b = c.bin0(v[k]);
                if (valid(v[k])) s.add(b, 0, true);
            }
        });
        j = join(s, true);
        const int k = (int)min(j.total, (u64)o.top_k);
        find(s, j, (u64)k, 0);
        const int bin = s.cut[0].bin;
        const u64 nc = s.cut[0].before + s.cut[0].sum;
        if (nc <= SR_CAP) {
            // few enough ids down to the k-th's bin: CTA 0 ends the row with them
            gather(s, c, true, [&](float v) { return c.bin0(v) <= bin; }, [](uint32_t, uint32_t) { return true; });
            if (rank == 0) finish_list(s, (int)nc, k, o, ids + row);
            return;
        }
        if (j.total > (u64)o.top_k) {
            cluster_sync();                 // (s.cut has been read)
            const Item it = select(s, j, (u64)k, true);
            if (tid == 0) {
                s.c.k_key = it.key;
                s.c.k_id = it.id;
                s.c.has_k = 1;
            }
        }
        __syncthreads();
    } else if (!sorted) {
        // id order: thread t has ids t per .. (an odd stride, so that a warp's reads fall in different banks)
        __syncthreads();
        const int per = ((n + SR_THREADS - 1) / SR_THREADS) | 1;
        const int i0 = min(n, tid * per), i1 = min(n, i0 + per);
        const RowConst c = s.c;
        const float* xs = s.xs;
        u64 sum = 0, mine;
#pragma unroll 4
        for (int i = i0; i < i1; ++i) sum += c.mass(c.prob(xs[i], s.exp2_table));
        u64 before = block_before(s, sum, &mine);
        if (tid < C) *remote(&s.part[rank], tid) = mine;
        cluster_sync();
        u64 total = 0;
        for (int r = 0; r < C; ++r) {
            if (r < rank) before += s.part[r];
            total += s.part[r];
        }
        const u64 target = share_of(o.draw, total);
        if (before < target && before + sum >= target) {
            for (int i = i0; i < i1; ++i) {
                before += c.mass(c.prob(xs[i], s.exp2_table));
                if (before >= target) {
                    ids[row] = id0 + i;
                    break;
                }
            }
        }
        return;
    }
    // masses: below 2^-(F+1) of the largest nothing is left, so the histogram's range ends there
    if (tid == 0) s.c.inv_w = width(fminf(half_range, (float)fmin((frac + 2) * 0.6931471805599453 * o.temperature * 0.5, (double)FLT_MAX)));
    clear_hist(s);
    const RowConst c = s.c;
    u64 over = 0;                           // the sum of the kept ids with p >= min_p
    const double min_p = o.min_p;
    each_four(s, [&](int i, const float (&v)[4]) {
        double p[4];
        u64 m[4];
        int b[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            p[k] = c.prob(v[k], s.exp2_table);
            b[k] = c.bin0(v[k]);
            m[k] = c.has_k && !c.kept(order_key(v[k]), (uint32_t)(id0 + i + k)) ? 0ull : c.mass(p[k]);
            over += p[k] >= min_p ? m[k] : 0ull;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (m[k]) s.add(b[k], m[k], false);
    });
    if (o.min_p > 0.0) {
        u64 mine;
        block_before(s, over, &mine);
        if (tid < C) *remote(&s.min_part[rank], tid) = mine;
    }
    j = join(s, false);
    over = ~0ull;
    if (o.min_p > 0.0) {
        over = 0;
        for (int r = 0; r < C; ++r) over += s.min_part[r];
    }
    // the nucleus's last bin, then the bins that the pick falls in whatever id of that bin ends the nucleus
    int nb = -1;
    u64 nbefore = 0, ntarget = 0, s_lo = j.total, s_hi = j.total;
    if (o.top_p < 1.0) {
        ntarget = share_of(o.top_p, j.total);
        find(s, j, ntarget, 0);
        nb = s.cut[0].bin;
        nbefore = s.cut[0].before;
        s_lo = nbefore + 1;
        s_hi = nbefore + s.cut[0].sum;
    }
    const u64 t_lo = share_of(o.draw, max(1ull, min(s_lo, over))), t_hi = share_of(o.draw, max(1ull, min(s_hi, over)));
    const uint32_t hi_in = __ballot_sync(0xffffffffu, j.before < t_hi && j.before + j.v >= t_hi);
    if (hi_in && (tid & 31) < C) remote(&s.cut[1], tid & 31)->bin_hi = rank * (s.bins / C) + (tid & ~31) + __ffs(hi_in) - 1;
    find(s, j, t_lo, 0, 1);
    const int p_lo = s.cut[1].bin, p_hi = s.cut[1].bin_hi;
    const u64 pbefore = s.cut[1].before;
    gather(s, c, false, [&](float v) {
        const int b = c.bin0(v);
        return b == nb || (b >= p_lo && b <= p_hi);
    }, [](uint32_t, uint32_t) { return true; });
    const int nc = remote(&s, 0)->n_cand;
    // CTA 0 ends the row; it leaves once the others have read its count
    cluster_arrive();
    if (nc <= SR_CAP) {
        if (rank == 0) finish_bins(s, nc, nb, nbefore, ntarget, p_lo, p_hi, pbefore, j.total, over, o.draw, ids + row);
        cluster_wait();
        return;
    }
    cluster_wait();
    // crowded bins: one cut after the other
    u64 sum = j.total;
    if (nb >= 0) sum = select(s, j, ntarget, false).cum;
    sum = max(1ull, min(sum, over));
    const Item it = select(s, j, share_of(o.draw, sum), false);
    if (lead) ids[row] = (int32_t)it.id;
}

// CTAs a row: one for every 8192 logits, up to 8.
int cluster_for(int V)
{
    int c = 1;
    while (c < SR_MAX_CLUSTER && V > 8192 * c) c *= 2;
    return c;
}

}  // namespace

void sample_rows(const float* logits, int64_t ld, int V, int rows, const wl_sample_opts* opts, int32_t* ids, cudaStream_t s)
{
    if (rows <= 0) return;
    const int C = cluster_for(V);
    const int slice = (int)((((int64_t)V + C - 1) / C + 3) / 4 * 4);
    const bool in_smem = slice <= SR_SLICE_MAX;
    const size_t smem = (sizeof(Row) + 15) / 16 * 16 + (in_smem ? (size_t)slice * 4 : 0);
    int bits = 0;
    while ((1ll << bits) < V) ++bits;
    // (the limit is the function's, not the launch's: the largest of all vocabularies, so that no other thread's call lowers it
    // between this one's limit and its launch)
    static std::atomic<bool> done[64];
    ensure_smem_attr(k_sample_rows, (int)((sizeof(Row) + 15) / 16 * 16 + SR_SLICE_MAX * 4), done);
    for (int r0 = 0; r0 < rows; r0 += 65535) {
        launch_cluster(k_sample_rows, dim3(C, std::min(rows - r0, 65535)), dim3(SR_THREADS), smem, s, C, logits + (int64_t)r0 * ld, ld, V,
                       std::min(51, 62 - bits), opts + r0, ids + r0, slice, in_smem ? 1 : 0);
        note_launch();
    }
}

}  // namespace k
}  // namespace wl
