// Device code shared by the kernels of the 4-bit KV cache (wl_kv4.cu, wl_kv4_mma.cu): the cache's layout, the codes' way into
// fp16, visible positions, and the join of ranges.
#pragma once
#include <cfloat>
#include <climits>
#include <cstdint>
#include <cuda_fp16.h>
#include "wl_common.h"
#include "wl_kernels.h"
#include "wl_launch.cuh"
#include "wl_mma.cuh"

namespace wl {
namespace k {

// Cache of row t: its base pointer (a RowKV with a layer offset, or a bare array of pointers).
struct Kv4Rows {
    const uint8_t* p;
    int pitch, layer;
    __device__ __forceinline__ uint8_t* base(int t) const
    {
        const uint8_t* e = p + (int64_t)t * pitch;
        uint8_t* b = *reinterpret_cast<uint8_t* const*>(e);
        if (pitch == (int)sizeof(RowKV)) b += (int64_t)layer * reinterpret_cast<const RowKV*>(e)->layer_stride * 2;
        return b;
    }
};

struct Kv4Att {
    const float* q;
    float* out;
    Kv4Rows rows;
    const int32_t* pos;
    int64_t capacity;
    int T, R, heads, kv_heads, S, s_max;    // S: ranges a row may be cut into (the stride of the partials)
    int alone;                              // rows of up to this many ranges are walked by one CTA
    float scale;
    int window, sinks;
    float* part;                            // [T][heads][S][HD]
    float* ml;                              // [T][heads][S][2]: maximum (log2 units), sum
    int* tickets;
    int* err;
};

// wl_kv4_mma.cu's kernel (head_dim 64 and 128): q_blocks CTAs of 128 queries a run and KV head (an even number of pairs'), a.S
// ranges each.
void kv4_attention_mma(const Kv4Att& a, int head_dim, int q_blocks, bool pairs, cudaStream_t s);

namespace {

constexpr int KV4_P = 16;                   // positions per tile
constexpr int kv4_tile_bytes(int HD) { return 18 * HD; }

// A row's state: 0 live, 1 padding (position < 0: nothing is read or written for it), 2 refused (a position past the
// cache, a null or misaligned cache).
__device__ __forceinline__ int kv4_row_state(const uint8_t* base, int64_t p, int64_t capacity)
{
    if (p < 0) return 1;
    return p >= capacity || !base || ((uintptr_t)base & 15) ? 2 : 0;
}

// Word index of (half, lane, block) in a code area.
template <int HD> __device__ __forceinline__ int kv4_word(int half, int lane, int b)
{
    constexpr int NB = HD / 32, W = NB < 4 ? NB : 4;
    return (b >> 2) * 256 + (half * 32 + lane) * W + (b & 3);
}

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// D = A B and D += A B for m16n8k16 in fp16 with fp32 sums.
__device__ __forceinline__ void mma_zero(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_add(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

// (w & mask) | bits in one instruction.
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t bits)
{
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "r"(mask), "r"(bits));
    return r;
}

// Eight codes to four fp16 pairs of c - 8: nibbles (0, 4), (1, 5), (2, 6), (3, 7). A nibble below 1024's exponent is
// 1024 + c, or 1024 + 16 c four bits up.
__device__ __forceinline__ void unpack_signed(uint32_t w, uint32_t (&r)[4])
{
    const __half2 m1032 = __floats2half2_rn(1032.f, 1032.f), s16 = __floats2half2_rn(0.0625f, 0.0625f),
                  m72 = __floats2half2_rn(-72.f, -72.f);
    const uint32_t w8 = w >> 8;
    r[0] = h2_bits(__hsub2(bits_h2(and_or(w, 0x000F000Fu, 0x64006400u)), m1032));
    r[1] = h2_bits(__hfma2(bits_h2(and_or(w, 0x00F000F0u, 0x64006400u)), s16, m72));
    r[2] = h2_bits(__hsub2(bits_h2(and_or(w8, 0x000F000Fu, 0x64006400u)), m1032));
    r[3] = h2_bits(__hfma2(bits_h2(and_or(w8, 0x00F000F0u, 0x64006400u)), s16, m72));
}

// Pairs of floats in one instruction.
__device__ __forceinline__ uint64_t f2(float lo, float hi)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 unf2(uint64_t v)
{
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// fp16 roundings of a pair and of what they leave.
__device__ __forceinline__ void split_h2(uint64_t ab, uint32_t& hi, uint32_t& lo)
{
    const float2 v = unf2(ab);
    const __half2 h = __floats2half2_rn(v.x, v.y);
    const float2 f = __half22float2(h);
    const float2 d = unf2(fma2(f2(f.x, f.y), f2(-1.f, -1.f), ab));
    hi = h2_bits(h);
    lo = h2_bits(__floats2half2_rn(d.x, d.y));
}

// The same with the remainders times 2^11: a remainder is 2^-11 of its value at most, so it is brought to the value's size, and
// keeps its bits where the value is near fp16's smallest (for remainders whose products have sums of their own).
constexpr float REM_UP = 2048.f;
__device__ __forceinline__ void split_h2_up(uint64_t ab, uint32_t& hi, uint32_t& lo)
{
    const float2 v = unf2(ab);
    const __half2 h = __floats2half2_rn(v.x, v.y);
    const float2 f = __half22float2(h);
    const float2 d = unf2(mul2(fma2(f2(f.x, f.y), f2(-1.f, -1.f), ab), f2(REM_UP, REM_UP)));
    hi = h2_bits(h);
    lo = h2_bits(__floats2half2_rn(d.x, d.y));
}

// The words of one lane's fragments: NB consecutive (planes of 4) 32-bit words.
template <int HD> __device__ __forceinline__ void lane_words(const uint8_t* area, int half, int lane, uint32_t (&w)[HD / 32])
{
    constexpr int NB = HD / 32;
    const uint32_t* p = reinterpret_cast<const uint32_t*>(area);
    if constexpr (NB == 2) {
        const uint2 x = lds64(p + (half * 32 + lane) * 2);
        w[0] = x.x; w[1] = x.y;
    } else if constexpr (NB == 3) {
#pragma unroll
        for (int b = 0; b < 3; ++b) w[b] = p[(half * 32 + lane) * 3 + b];
    } else {
#pragma unroll
        for (int pl = 0; pl < NB / 4; ++pl) {
            const uint4 x = lds128(p + pl * 256 + (half * 32 + lane) * 4);
            w[4 * pl] = x.x; w[4 * pl + 1] = x.y; w[4 * pl + 2] = x.z; w[4 * pl + 3] = x.w;
        }
    }
}

// The scales of positions r, r + 1 (r even): NB fp16 pairs' words, position-major.
template <int HD> __device__ __forceinline__ void lane_scales(const uint8_t* area, int r, uint32_t (&w)[HD / 32])
{
    constexpr int NB = HD / 32;
    const uint32_t* p = reinterpret_cast<const uint32_t*>(area) + r * NB / 2;
    if constexpr (NB == 2) {
        const uint2 x = lds64(p);
        w[0] = x.x; w[1] = x.y;
    } else if constexpr (NB == 3) {
#pragma unroll
        for (int b = 0; b < 3; ++b) w[b] = p[b];
    } else {
#pragma unroll
        for (int i = 0; i < NB / 4; ++i) {
            const uint4 x = lds128(p + 4 * i);
            w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w;
        }
    }
}
// Scale b of position e (0, 1) of those words.
template <int NB> __device__ __forceinline__ float scale_of(const uint32_t (&w)[NB], int e, int b)
{
    const int i = e * NB + b;
    const float2 f = __half22float2(bits_h2(w[i >> 1]));
    return i & 1 ? f.y : f.x;
}

// One query's visible positions: j < n and (j >= first or j < sink).
struct Vis {
    int n, first, sink;
    __device__ __forceinline__ bool operator()(int j) const { return j < n && (j >= first || j < sink); }
};
__device__ __forceinline__ Vis visible(int p, int window, int sinks)
{
    const int n = p + 1, first = window > 0 && n > window ? n - window : 0;
    return Vis{n, first, min(sinks, first)};
}

// The tiles that hold positions of [0, sink) or [first, n): item i of the list is tile i below head, else i + skip.
struct TileList {
    int head, skip, count;
    __device__ __forceinline__ int at(int i) const { return i < head ? i : i + skip; }
};
__device__ __forceinline__ TileList tile_list(int n, int first, int sink)
{
    const int t1 = first >> 4, head = min((sink + 15) >> 4, t1), last = (n - 1) >> 4;
    return TileList{head, t1 - head, n > 0 ? head + last - t1 + 1 : 0};
}


// A running maximum is followed only when it is passed by a factor 2^6: weights up to 2^6 cost nothing, and the output's
// sums are rescaled a few times a row and not at most tiles.
constexpr float ATT_SLACK = 6.f;

constexpr int ATT_MAX_RANGES = 96;          // ranges a row may be cut into

// A row's ranges are joined one after the other: (M, L, o) and the next range's (m, l, p) give M' = max(M, m),
// L e^(M - M') + l e^(m - M') and the same of o. The order and the operations are the same whether one CTA walks all ranges
// (JoinState) or the last of several CTAs joins what the others left (join_ranges), so a row's bits are too.
struct JoinState {
    float M, L;
    float4 o;
    __device__ __forceinline__ void add(float m, float l, const float4& p, bool first)
    {
        if (first) {
            M = m;
            L = l;
            o = p;
            return;
        }
        const float mn = fmaxf(M, m), mu = mn == -INFINITY ? 0.f : mn, a = ex2(M - mu), b = ex2(m - mu);
        M = mn;
        L = __fmaf_rn(l, b, __fmul_rn(L, a));
        o.x = __fmaf_rn(p.x, b, __fmul_rn(o.x, a));
        o.y = __fmaf_rn(p.y, b, __fmul_rn(o.y, a));
        o.z = __fmaf_rn(p.z, b, __fmul_rn(o.z, a));
        o.w = __fmaf_rn(p.w, b, __fmul_rn(o.w, a));
    }
    __device__ __forceinline__ float4 out() const
    {
        const float inv = L != 0.f ? __fdiv_rn(1.f, L) : 0.f;      // (a NaN sum stays NaN; no visible position: zeros)
        return make_float4(__fmul_rn(o.x, inv), __fmul_rn(o.y, inv), __fmul_rn(o.z, inv), __fmul_rn(o.w, inv));
    }
};

// Where the queries of a join are: query i is at (row, head) index base + (q0 + i) / G * heads + (q0 + i) % G.
struct RowMap {
    int64_t base;
    int q0, G, heads;
    __device__ __forceinline__ int64_t at(int i) const { return base + (int64_t)((q0 + i) / G) * heads + (q0 + i) % G; }
};

// Joins the n ranges (of S places for partials) of nh queries, by a CTA of NT threads: a warp takes a head's
// factors at a time (the running maxima by a scan), then every thread 4 output values, its loads of 8 ranges in flight
// together. w: nh * (3 n + 1) floats of shared memory.
template <int HD, int NT>
__device__ __noinline__ void join_ranges(const float* ml_, const float* part, float* out, int S, int nh, int n, float* w, RowMap row)
{
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (n <= 8) {
        // few ranges: every thread makes the factors of its output values itself
        for (int i = threadIdx.x; i < nh * (HD / 4); i += NT) {
            const int64_t at = row.at(i / (HD / 4));
            const int d = i % (HD / 4) * 4;
            const float2* ml = reinterpret_cast<const float2*>(ml_) + at * S;
            const float4* pp = reinterpret_cast<const float4*>(part + at * S * HD + d);
            float2 x[8];
            float4 p[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k < n) {
                    x[k] = __ldcg(ml + k);
                    p[k] = __ldcg(pp + (int64_t)k * (HD / 4));
                }
            JoinState j;
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k < n) j.add(x[k].x, x[k].y, p[k], k == 0);
            *reinterpret_cast<float4*>(out + at * HD + d) = j.out();
        }
        return;
    }
    for (int h = warp; h < nh; h += NT / 32) {
        const float2* ml = reinterpret_cast<const float2*>(ml_) + row.at(h) * S;
        float* wh = w + h * (3 * n + 1);    // of range s: what the ranges before it are scaled by, what it is, its sum
        float M = -INFINITY;                // the maximum of the ranges before this lane's
#pragma unroll
        for (int i = 0; i < ATT_MAX_RANGES / 32; ++i) {
            if (32 * i >= n) break;
            const int s = lane + 32 * i;
            const float2 x = s < n ? __ldcg(ml + s) : make_float2(-INFINITY, 0.f);
            float inc = x.x;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const float y = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc = fmaxf(inc, y);
            }
            float before = __shfl_up_sync(0xffffffffu, inc, 1);
            before = lane ? fmaxf(before, M) : M;
            const float mn = fmaxf(before, x.x), mu = mn == -INFINITY ? 0.f : mn;
            if (s < n) {
                wh[3 * s] = ex2(before - mu);
                wh[3 * s + 1] = ex2(x.x - mu);
                wh[3 * s + 2] = x.y;
            }
            M = fmaxf(M, __shfl_sync(0xffffffffu, inc, 31));
        }
        __syncwarp();
        float L = wh[2];
#pragma unroll 8
        for (int s = 1; s < n; ++s) L = __fmaf_rn(wh[3 * s + 2], wh[3 * s + 1], __fmul_rn(L, wh[3 * s]));
        __syncwarp();
        if (lane == 0) wh[3 * n] = L != 0.f ? __fdiv_rn(1.f, L) : 0.f;      // (as JoinState::out)
    }
    __syncthreads();
    for (int i = threadIdx.x; i < nh * (HD / 4); i += NT) {
        const int h = i / (HD / 4), d = i % (HD / 4) * 4;
        const float4* pp = reinterpret_cast<const float4*>(part + row.at(h) * S * HD + d);
        const float* wh = w + h * (3 * n + 1);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int s0 = 0; s0 < n; s0 += 8) {
            float4 p[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) p[k] = s0 + k < n ? __ldcg(pp + (int64_t)(s0 + k) * (HD / 4)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int s = s0 + k;
                if (s >= n) break;
                const float fa = wh[3 * s], fb = wh[3 * s + 1];
                o.x = s ? __fmaf_rn(p[k].x, fb, __fmul_rn(o.x, fa)) : p[k].x;
                o.y = s ? __fmaf_rn(p[k].y, fb, __fmul_rn(o.y, fa)) : p[k].y;
                o.z = s ? __fmaf_rn(p[k].z, fb, __fmul_rn(o.z, fa)) : p[k].z;
                o.w = s ? __fmaf_rn(p[k].w, fb, __fmul_rn(o.w, fa)) : p[k].w;
            }
        }
        const float inv = wh[3 * n];
        *reinterpret_cast<float4*>(out + row.at(h) * HD + d) =
            make_float4(__fmul_rn(o.x, inv), __fmul_rn(o.y, inv), __fmul_rn(o.z, inv), __fmul_rn(o.w, inv));
    }
}

// After a wait gave up: what is still in flight ends before the CTA does (bounded as well).
__device__ __forceinline__ void mbar_drain(uint64_t* bar, uint32_t parity)
{
    const unsigned long long t0 = globaltimer_ns();
    while (!mbar_try_wait(bar, parity) && globaltimer_ns() - t0 <= MBAR_WAIT_NS) {
    }
}

// Takes a ticket after the CTA's partials; true in the CTA that took the last of n.
__device__ __forceinline__ bool last_ticket(int* ctr, int n)
{
    __shared__ int last;
    __syncthreads();
    if (threadIdx.x == 0) {
        int ticket;
        asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(ticket) : "l"(ctr) : "memory");
        last = ticket == n - 1;
        if (last) *ctr = 0;
    }
    __syncthreads();
    return last;
}

}  // namespace

}  // namespace k
}  // namespace wl
