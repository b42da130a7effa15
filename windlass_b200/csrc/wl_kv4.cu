// The 4-bit KV cache: rotary append, read-back and attention (whole context, or a sliding window with sinks).
//
// Values. A key or value head is cut into blocks of 32. A block keeps an fp16 scale d = m / -8, m its value of largest
// magnitude (the positive one of a pair), and 32 codes c = clamp(floor(x / d + 8.5), 0, 15); it stands for (c - 8) d
// (the values of a Q4_0 block). A block that holds an infinity or a NaN gets d = NaN and reads as NaN.
//
// Layout. A cache is an array of tiles [position / 16][kv head], each 18 * HD bytes: the keys' codes (8 HD bytes), the
// values' codes (8 HD), the keys' scales [16][HD / 32] and the values' scales [16][HD / 32]. One 1-D bulk copy brings a
// tile, and the codes lie in the order in which the MMA fragments read them, so that a lane's 16-byte shared-memory
// loads are its fragments and nothing is shuffled. With NB = HD / 32 blocks and W = min(4, NB), a code area is planes
// of 4 blocks, each [half][lane = 4 g + c][W] 32-bit words:
//   keys:   word (half, g, c, b) = position 8 half + g, dims 32 b + 8 c + 0..7 in nibbles 0..7;
//   values: word (half, g, c, b) = positions 8 half + 2 c (low 16 bits) and + 1 (high), dims 32 b + 4 g + 0..3.
//
// Attention. The query heads of one KV head share its codes: a tile of 8 queries (heads of a row, or rows of a prompt)
// is the 16-row side of m16n8k16 MMAs, each query twice: rows 0-7 its values' fp16 roundings, rows 8-15 what the
// roundings left (together 22 bits of the row's largest value). Keys and values enter as fp16 integers -8..7. (Keys as
// fp16 subnormals, their codes cut out by a mask, with 8 times the query's sum taken off, took 4 % less time and lost bits in
// the MMA's sums: 2.3e-6 to 2.8e-6 of the output, against 2.5e-7 to 4.3e-7 so.) All products are exact, sums are fp32; the
// block scales are applied outside: to each block's fp32 sums for the scores, and to the weights before they are split
// for the values (p * d, per block, times a power of two vs for fp16's range). fp16 has no steps below 2^-24, so the remainders
// of those weights enter times 2^11 (their products have sums of their own): 22 bits down to p d = 2^-14 / vs, and at most
// 2^-36 / vs lost below. vs is 2^8 where no value's scale reaches 2, so that is 2^-44 beside weights of up to 1, and a
// position 26 nats below the largest still counts. (Without the 2^11, positions 15 nats below a sink lost a tenth of
// their weight where the values are small; it costs 2 % of a row's time.)
#include <algorithm>
#include "wl_kv4.cuh"

namespace wl {
namespace k {

namespace {

// ------------------------------------------------------------------------------------------------------------------
// append and read
// ------------------------------------------------------------------------------------------------------------------
// q's part: a thread turns 4 consecutive dims (or, with NEOX pairs, 4 and their 4 partners), APP_Q such units, its loads in
// flight together. k's and v's part: a thread owns 8 consecutive dims of one head; four threads a block of 32. The rotation
// of k and the codes are computed in 64 bits: a code's border is a step of the value, so a difference in the last bit of
// 32 would decide codes, and 64-bit arithmetic costs nothing here (about 30 operations a value against the bytes a row
// moves). VEC: rope_dims is a multiple of 16 and the table 16-byte aligned, so that pairs, partners and angles come in
// 16-byte loads; otherwise one by one.
// Measured: one row of 64 heads on 8 of 128 dims 3.5 us, 61 rows of 32 on 4 4.8 us (both a launch's latency), 2048 rows of 64
// on 8 43.8 us: 165 MB, 3.8 TB/s, 0.58 of a copy's rate. Bound there by the loads in flight: q's part alone is a copy.
constexpr int APP_Q = 4;

// 4 dims from d of a head's row x into y: rotated (the pairs' first dims of NEOX: both), or copied.
template <bool VEC>
__device__ __forceinline__ void rotate4(const float* x, float* y, const float* cs, int d, int rope_dims, bool neox, bool copy)
{
    const int half = rope_dims / 2;
    if (d >= rope_dims) {
        if (copy) *reinterpret_cast<float4*>(y + d) = *reinterpret_cast<const float4*>(x + d);
    } else if (VEC && !neox) {
        const float4 v = *reinterpret_cast<const float4*>(x + d), t = *reinterpret_cast<const float4*>(cs + d);
        float4 o;
        o.x = __fsub_rn(__fmul_rn(v.x, t.x), __fmul_rn(v.y, t.y));
        o.y = __fadd_rn(__fmul_rn(v.x, t.y), __fmul_rn(v.y, t.x));
        o.z = __fsub_rn(__fmul_rn(v.z, t.z), __fmul_rn(v.w, t.w));
        o.w = __fadd_rn(__fmul_rn(v.z, t.w), __fmul_rn(v.w, t.z));
        *reinterpret_cast<float4*>(y + d) = o;
    } else if (VEC) {
        if (d >= half) return;              // (the first dims' thread writes both)
        const float4 v = *reinterpret_cast<const float4*>(x + d), u = *reinterpret_cast<const float4*>(x + d + half);
        const float4 t0 = *reinterpret_cast<const float4*>(cs + 2 * d), t1 = *reinterpret_cast<const float4*>(cs + 2 * d + 4);
        float4 o, w;
        o.x = __fsub_rn(__fmul_rn(v.x, t0.x), __fmul_rn(u.x, t0.y));
        w.x = __fadd_rn(__fmul_rn(v.x, t0.y), __fmul_rn(u.x, t0.x));
        o.y = __fsub_rn(__fmul_rn(v.y, t0.z), __fmul_rn(u.y, t0.w));
        w.y = __fadd_rn(__fmul_rn(v.y, t0.w), __fmul_rn(u.y, t0.z));
        o.z = __fsub_rn(__fmul_rn(v.z, t1.x), __fmul_rn(u.z, t1.y));
        w.z = __fadd_rn(__fmul_rn(v.z, t1.y), __fmul_rn(u.z, t1.x));
        o.w = __fsub_rn(__fmul_rn(v.w, t1.z), __fmul_rn(u.w, t1.w));
        w.w = __fadd_rn(__fmul_rn(v.w, t1.w), __fmul_rn(u.w, t1.z));
        *reinterpret_cast<float4*>(y + d) = o;
        *reinterpret_cast<float4*>(y + d + half) = w;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int d0 = d + e;
            if (d0 >= rope_dims) {
                if (copy) y[d0] = x[d0];
                continue;
            }
            // the thread of a pair's first dim writes both, so that rotating in place never reads a rotated value
            if (neox ? d0 >= half : d0 & 1) continue;
            const int i = neox ? d0 : d0 >> 1, d1 = neox ? d0 + half : d0 + 1;
            const float c = cs[2 * i], sn = cs[2 * i + 1], x0 = x[d0], x1 = x[d1];
            y[d0] = __fsub_rn(__fmul_rn(x0, c), __fmul_rn(x1, sn));
            y[d1] = __fadd_rn(__fmul_rn(x0, sn), __fmul_rn(x1, c));
        }
    }
}

template <int HD, bool VEC>
__global__ void __launch_bounds__(128, 8) k_kv4_append(const float* q, float* q_out, const float* k, const float* v, int T,
                                                       int heads, int kv_heads, const float* table, int rope_dims, int neox,
                                                       Kv4Rows rows, const int32_t* pos, int64_t capacity, int kv_blocks)
{
    constexpr int CH = HD / 8;              // 8-dim chunks of a head
    pdl_trigger();
    pdl_wait();
    const int half = rope_dims / 2;
    for (int t = blockIdx.y; t < T; t += gridDim.y) {
        const int p = pos[t];
        uint8_t* base = rows.base(t);
        if (kv4_row_state(base, p, capacity)) continue;
        const float* cs = table + (int64_t)p * rope_dims;
        if ((int)blockIdx.x >= kv_blocks) {
            const int u0 = ((int)blockIdx.x - kv_blocks) * 128 * APP_Q + threadIdx.x;
            const float* x = q + (int64_t)t * heads * HD;
            float* y = q_out + (int64_t)t * heads * HD;
#pragma unroll
            for (int i = 0; i < APP_Q; ++i) {
                const int u = u0 + 128 * i, h = u / (HD / 4);
                if (h < heads) rotate4<VEC>(x + h * HD, y + h * HD, cs, u % (HD / 4) * 4, rope_dims, neox != 0, q_out != q);
            }
            continue;
        }
        const int u = blockIdx.x * 128 + threadIdx.x;
        const int units = kv_heads * CH;
        const bool live = u < 2 * units, is_v = u >= units;
        const int uu = live ? (is_v ? u - units : u) : 0;
        const int h = uu / CH, d0 = uu % CH * 8;
        const float* x = (is_v ? v : k) + ((int64_t)t * kv_heads + h) * HD;
        float xf[8];
        *reinterpret_cast<float4*>(xf) = *reinterpret_cast<const float4*>(x + d0);
        *reinterpret_cast<float4*>(xf + 4) = *reinterpret_cast<const float4*>(x + d0 + 4);
        double xd[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) xd[e] = xf[e];
        if (!is_v && d0 < rope_dims) {
            // products of 24-bit factors are exact in 53 bits, so one rounding follows, with or without fma
            if (VEC && neox) {
                const bool first = d0 < half;
                const int i0 = first ? d0 : d0 - half;
                const float* o = x + (first ? d0 + half : d0 - half);
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float4 t2 = *reinterpret_cast<const float4*>(cs + 2 * (i0 + e));
                    const float2 o2 = *reinterpret_cast<const float2*>(o + e);
                    xd[e] = first ? xd[e] * t2.x - (double)o2.x * t2.y : (double)o2.x * t2.y + xd[e] * t2.x;
                    xd[e + 1] = first ? xd[e + 1] * t2.z - (double)o2.y * t2.w : (double)o2.y * t2.w + xd[e + 1] * t2.z;
                }
            } else if (VEC) {
#pragma unroll
                for (int e = 0; e < 8; e += 4) {
                    const float4 t2 = *reinterpret_cast<const float4*>(cs + d0 + e);
                    const double a = xd[e], b = xd[e + 1], g = xd[e + 2], r = xd[e + 3];
                    xd[e] = a * t2.x - b * t2.y;
                    xd[e + 1] = a * t2.y + b * t2.x;
                    xd[e + 2] = g * t2.z - r * t2.w;
                    xd[e + 3] = g * t2.w + r * t2.z;
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int d = d0 + e;
                    if (d >= rope_dims) continue;
                    const bool first = neox ? d < half : (d & 1) == 0;
                    const int i = neox ? (first ? d : d - half) : d >> 1;
                    const double c = cs[2 * i], sn = cs[2 * i + 1];
                    const double o = neox ? (double)x[first ? d + half : d - half] : (double)xf[e ^ 1];
                    xd[e] = first ? xd[e] * c - o * sn : o * sn + xd[e] * c;
                }
            }
        }
        double hi = xd[0], lo = xd[0];
        bool bad = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            hi = xd[e] > hi ? xd[e] : hi;
            lo = xd[e] < lo ? xd[e] : lo;
            bad |= !(fabs(xd[e]) <= 1.7e308);
        }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            const double a = __shfl_xor_sync(0xffffffffu, hi, o), b = __shfl_xor_sync(0xffffffffu, lo, o);
            hi = a > hi ? a : hi;
            lo = b < lo ? b : lo;
        }
        bad = (__ballot_sync(0xffffffffu, bad) >> (threadIdx.x & 28)) & 15u;
        const double m = hi >= -lo ? hi : lo;
        float df = (float)(m / -8.0);
        df = fminf(fmaxf(df, -65504.f), 65504.f);       // a scale past fp16's largest saturates
        const __half dh = bad ? __ushort_as_half((unsigned short)0x7e00) : __float2half_rn(df);
        const double dd = (double)__half2float(dh), inv = dd != 0.0 ? 1.0 / dd : 0.0;
        uint32_t w = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const double c = floor(__dadd_rn(__dmul_rn(xd[e], inv), 8.5));
            w |= (uint32_t)(c >= 15.0 ? 15 : c > 0.0 ? (int)c : 0) << (4 * e);      // (a NaN gives 0)
        }
        if (!live) continue;
        uint8_t* tile = base + ((int64_t)(p >> 4) * kv_heads + h) * kv4_tile_bytes(HD);
        const int b = d0 >> 5, c4 = d0 >> 3 & 3, r = p & 15;
        if (!is_v) {
            reinterpret_cast<uint32_t*>(tile)[kv4_word<HD>(r >> 3, (r & 7) * 4 + c4, b)] = w;
        } else {
            // dims 8 c4 .. +3 and + 4 .. +7 are g = 2 c4 and 2 c4 + 1
            uint16_t* vw = reinterpret_cast<uint16_t*>(tile + 8 * HD);
            const int lane = (r & 7) >> 1;
            vw[2 * kv4_word<HD>(r >> 3, 8 * c4 + lane, b) + (r & 1)] = (uint16_t)w;
            vw[2 * kv4_word<HD>(r >> 3, 8 * c4 + 4 + lane, b) + (r & 1)] = (uint16_t)(w >> 16);
        }
        if (c4 == 0)
            reinterpret_cast<__half*>(tile + (is_v ? 17 : 16) * HD)[r * (HD / 32) + b] = dh;
    }
}

// The fp16 values that position pos[t] of row t's cache stands for; zeros for a padding row, NaN for a refused one.
template <int HD>
__global__ void __launch_bounds__(128) k_kv4_read(Kv4Rows rows, const int32_t* pos, int T, int kv_heads, int64_t capacity,
                                                  __half* k_out, __half* v_out)
{
    constexpr int CH = HD / 8;
    pdl_trigger();
    pdl_wait();
    const int units = kv_heads * CH;
    const int u = blockIdx.x * 128 + threadIdx.x;
    if (u >= 2 * units) return;
    const bool is_v = u >= units;
    const int uu = is_v ? u - units : u, h = uu / CH, d0 = uu % CH * 8, b = d0 >> 5, c4 = d0 >> 3 & 3;
    for (int t = blockIdx.y; t < T; t += gridDim.y) {
        const int p = pos[t];
        const uint8_t* base = rows.base(t);
        const int st = kv4_row_state(base, p, capacity);
        __half out[8];
        if (st) {
#pragma unroll
            for (int e = 0; e < 8; ++e) out[e] = st == 1 ? __half(__ushort_as_half((unsigned short)0)) : __half(__ushort_as_half((unsigned short)0x7e00));
        } else {
            const uint8_t* tile = base + ((int64_t)(p >> 4) * kv_heads + h) * kv4_tile_bytes(HD);
            const int r = p & 15;
            uint32_t w;
            if (!is_v) {
                w = reinterpret_cast<const uint32_t*>(tile)[kv4_word<HD>(r >> 3, (r & 7) * 4 + c4, b)];
            } else {
                const uint16_t* vw = reinterpret_cast<const uint16_t*>(tile + 8 * HD);
                const int lane = (r & 7) >> 1;
                w = (uint32_t)vw[2 * kv4_word<HD>(r >> 3, 8 * c4 + lane, b) + (r & 1)] |
                    (uint32_t)vw[2 * kv4_word<HD>(r >> 3, 8 * c4 + 4 + lane, b) + (r & 1)] << 16;
            }
            const float d = __half2float(reinterpret_cast<const __half*>(tile + (is_v ? 17 : 16) * HD)[r * (HD / 32) + b]);
#pragma unroll
            for (int e = 0; e < 8; ++e) out[e] = __float2half_rn((float)((int)(w >> (4 * e) & 15u) - 8) * d);
        }
        *reinterpret_cast<uint4*>((is_v ? v_out : k_out) + ((int64_t)t * kv_heads + h) * HD + d0) = *reinterpret_cast<uint4*>(out);
    }
}

// ------------------------------------------------------------------------------------------------------------------
// attention
// ------------------------------------------------------------------------------------------------------------------

// Running softmax of MT tiles of 8 queries: lane (g, c) keeps query g's reference maximum (in log2 units), its own share of
// the sum, and the output's fragments (o[.][0,1] the rows of the weights' roundings, [2,3] of what they left, times 2^11).
template <int HD, int MT> struct AttState {
    float m[MT], l[MT], o[MT][HD / 8][4];
    float vs;                   // the values' scales are multiplied by vs = 2^k, so that a weight's product stays below 2^15
    __device__ __forceinline__ void init()
    {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            m[i] = -INFINITY;
            l[i] = 0.f;
#pragma unroll
            for (int j = 0; j < HD / 8; ++j) o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.f;
        }
        vs = 256.f;
    }
    // Output fragment j's value e (0, 1), times vs.
    __device__ __forceinline__ float sum(int i, int j, int e) const { return fmaf(o[i][j][e + 2], 1.f / REM_UP, o[i][j][e]); }
};

// NT tiles of 16 positions (from positions tile0[.], one behind the other at sm) for MT query tiles. qf(i, b, s) gives the A
// fragment of query tile i, block b, step s (dims 32 b + 8 c + {2s, 2s + 4}, {2s + 1, 2s + 5} of lane c); ks undoes the
// queries' powers of two.
template <int HD, int MT, int NT, class QF>
__device__ __forceinline__ void kv4_tiles(const uint8_t* sm, int lane, const int (&tile0)[NT], const Vis (&vis)[MT], bool full,
                                          const QF& qf, const float (&ks)[MT], AttState<HD, MT>& st)
{
    constexpr int NB = HD / 32, TB = kv4_tile_bytes(HD);
    const int c = lane & 3;
    uint64_t s2[MT][2 * NT];                // scores of positions (2c, 2c + 1) and (2c + 8, 2c + 9), in the query's units
#pragma unroll
    for (int h = 0; h < 2 * NT; ++h) {
        const uint8_t* t = sm + h / 2 * TB;
        uint32_t kw[NB], dw[NB];
        lane_words<HD>(t, h & 1, lane, kw);
        lane_scales<HD>(t + 16 * HD, 8 * (h & 1) + 2 * c, dw);
#pragma unroll
        for (int i = 0; i < MT; ++i) s2[i][h] = f2(0.f, 0.f);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            uint32_t r[4];
            unpack_signed(kw[b], r);
            const uint64_t d01 = f2(scale_of<NB>(dw, 0, b), scale_of<NB>(dw, 1, b));
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                float d[4];
                mma_zero(d, qf(i, b, 0), r[0], r[1]);
                mma_add(d, qf(i, b, 1), r[2], r[3]);
                s2[i][h] = fma2(d01, add2(f2(d[0], d[1]), f2(d[2], d[3])), s2[i][h]);
            }
        }
    }
    uint32_t seen[MT], any_seen = 0u;       // bits (4 a tile) of the positions that this lane's queries see
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        if (!full) {
            seen[i] = 0u;
#pragma unroll
            for (int h = 0; h < 2 * NT; ++h) {
                float2 x = unf2(s2[i][h]);
                const int j = tile0[h / 2] + 2 * c + 8 * (h & 1);
                if (vis[i](j)) seen[i] |= 1u << (2 * h);
                else x.x = -INFINITY;
                if (vis[i](j + 1)) seen[i] |= 2u << (2 * h);
                else x.y = -INFINITY;
                s2[i][h] = f2(x.x, x.y);
            }
            any_seen |= seen[i];
        }
        float mx = -INFINITY;
#pragma unroll
        for (int h = 0; h < 2 * NT; ++h) {
            const float2 x = unf2(s2[i][h]);
            mx = fmaxf(mx, fmaxf(x.x, x.y));
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2)) * ks[i];
        if (__any_sync(0xffffffffu, mx > st.m[i] + ATT_SLACK)) {
            const float mn = mx > st.m[i] ? mx : st.m[i], a = st.m[i] == -INFINITY ? 0.f : ex2(st.m[i] - mn);
            st.l[i] *= a;
#pragma unroll
            for (int j = 0; j < HD / 8; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) st.o[i][j][e] *= a;
            st.m[i] = mn;
        }
        const float mu = st.m[i] == -INFINITY ? 0.f : st.m[i];
        const uint64_t k2 = f2(ks[i], ks[i]), m2 = f2(-mu, -mu);
#pragma unroll
        for (int h = 0; h < 2 * NT; ++h) {
            const float2 x = unf2(fma2(s2[i][h], k2, m2));
            const float p0 = ex2(x.x), p1 = ex2(x.y);
            st.l[i] += p0 + p1;
            s2[i][h] = f2(p0, p1);          // now the weights
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const uint8_t* t = sm + n * TB;
        uint32_t vd[2][NB], vw[2][NB];
        lane_scales<HD>(t + 17 * HD, 2 * c, vd[0]);
        lane_scales<HD>(t + 17 * HD, 2 * c + 8, vd[1]);
        if (!full) {
            // a position that no query of this lane sees may hold anything: its scales (perhaps NaN) count as zero
#pragma unroll
            for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                for (int i = 0; i < 2 * NB; ++i)
                    if (!(any_seen >> (4 * n + 2 * hf + i / NB) & 1u)) vd[hf][i >> 1] &= i & 1 ? 0x0000FFFFu : 0xFFFF0000u;
        }
        // scales below 2 need no care: 2 * 2^8 * (a weight up to 2^6) is 2^15. The exponent's top bit tells the others.
        uint32_t any = vd[0][0] | vd[1][0];
#pragma unroll
        for (int i = 1; i < NB; ++i) any |= vd[0][i] | vd[1][i];
        if (__any_sync(0xffffffffu, any & 0x40004000u)) {
            __half2 mx = __habs2(bits_h2(vd[0][0]));
#pragma unroll
            for (int i = 1; i < 2 * NB; ++i) mx = __hmax2(mx, __habs2(bits_h2(vd[i / NB][i % NB])));
            float a = fmaxf(__low2float(mx), __high2float(mx));
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
            if (a * st.vs > 512.f) {
                // larger scales than any so far: a smaller power of two, and the sums follow
                const float nv = ldexpf(1.f, max(8 - ilogbf(a), -7)), f = nv / st.vs;
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int j = 0; j < HD / 8; ++j)
#pragma unroll
                        for (int x = 0; x < 4; ++x) st.o[i][j][x] *= f;
                st.vs = nv;
            }
        }
        const __half2 v2 = __float2half2_rn(st.vs);
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
#pragma unroll
            for (int i = 0; i < NB; ++i) vd[hf][i] = h2_bits(__hmul2(bits_h2(vd[hf][i]), v2));
        lane_words<HD>(t + 8 * HD, 0, lane, vw[0]);
        lane_words<HD>(t + 8 * HD, 1, lane, vw[1]);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            uint32_t r0[4], r1[4];
            unpack_signed(vw[0][b], r0);
            unpack_signed(vw[1][b], r1);
            const uint64_t d01 = f2(scale_of<NB>(vd[0], 0, b), scale_of<NB>(vd[0], 1, b)),
                           d23 = f2(scale_of<NB>(vd[1], 0, b), scale_of<NB>(vd[1], 1, b));
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                uint4 a;
                uint64_t p01 = mul2(s2[i][2 * n], d01), p23 = mul2(s2[i][2 * n + 1], d23);
                if (MT > 1 && !full) {      // (a scale that only the lane's other queries see may be NaN)
                    const uint32_t see = seen[i] >> (4 * n);
                    const float2 x = unf2(p01), y = unf2(p23);
                    p01 = f2(see & 1u ? x.x : 0.f, see & 2u ? x.y : 0.f);
                    p23 = f2(see & 4u ? y.x : 0.f, see & 8u ? y.y : 0.f);
                }
                split_h2_up(p01, a.x, a.y);
                split_h2_up(p23, a.z, a.w);
#pragma unroll
                for (int j = 0; j < 4; ++j) mma_add(st.o[i][4 * b + j], a, r0[j], r1[j]);
            }
        }
    }
}

// The A fragments qa[b][s] of lane (g, c)'s query row (nullptr: zeros) and its terms. A power of two brings the row's largest
// value to 2^13..2^14, where fp16 and its remainder keep 22 bits.
template <int HD>
__device__ __forceinline__ void load_query(const float* x, int lane, float f, uint4 (&qa)[HD / 32][2], float& ks)
{
    constexpr int NB = HD / 32;
    const int c = lane & 3;
    float v[NB][8];
    float mx = 0.f;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        float4 lo = make_float4(0.f, 0.f, 0.f, 0.f), hi = lo;
        if (x) {
            lo = *reinterpret_cast<const float4*>(x + 32 * b + 8 * c);
            hi = *reinterpret_cast<const float4*>(x + 32 * b + 8 * c + 4);
        }
        const float y[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[b][e] = y[e] * f;
            mx = fmaxf(mx, fabsf(v[b][e]));
        }
    }
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    const int e = mx > 0.f && mx <= FLT_MAX ? min(100, 13 - ilogbf(mx)) : 0;      // (-114 at least)
    const float up = ldexpf(1.f, e);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            split_h2(f2(v[b][2 * s] * up, v[b][2 * s + 4] * up), qa[b][s].x, qa[b][s].y);
            split_h2(f2(v[b][2 * s + 1] * up, v[b][2 * s + 5] * up), qa[b][s].z, qa[b][s].w);
        }
    }
    ks = ldexpf(1.f, -e);
}

// A CTA of 8 warps, two an SM (128 registers, the queries' fragments in shared memory): against three CTAs of 4 warps with the
// fragments in registers, one row over 131000 positions 52.8 against 55.6 us (fewer ranges to join), 8 rows of up to 4100
// 15.5 against 19.1. A range holds 48 tiles at least: 6 to a warp.
constexpr int ATT_WARPS = 8;
constexpr int RUN_WARPS = 4;                // warps of a CTA of the runs' kernel
constexpr int ATT_TPS = 48;
constexpr int ATT_STAGES = 2;               // ring stages a warp, of two tiles each
constexpr int att_ctas(int HD) { return HD <= 128 ? 2 : 1; }

// Rows on their own (decode). A row's tiles are cut into ranges of att_range() tiles, from the row's own length; a CTA
// (range, KV head and tile of 8 query heads, row) gives a range's maximum, sum and output. Each warp streams its own tiles,
// every eighth pair of the range, through its ring of bulk copies, and the warps' sums are joined in warp order. The last
// CTA of a row joins the ranges, or, where there are rows enough to fill the SMs (ALONE: rows of up to a.alone ranges), one
// CTA walks a row's ranges: a row's bits do not depend on that, nor on the other rows.
// Measured: 64 heads on 8 of 128 dims over 131001 positions 57.9 us (151 MB, 2.6 TB/s, 0.40 of a copy's rate), 8 such rows of up
// to 4100 16.1 us, 64 rows of 32 on 8 behind a window of 1024 41.8 us (78 MB, 1.9 TB/s), 8 heads of 64 dims over 300
// positions 4.7 us. Bound by the warps' instructions: about 390 a tile of 16 positions and warp (the codes' masks, the scales'
// products, weights split in two), with the loads always two tiles ahead.
__device__ __forceinline__ int att_range(int tiles, int s_max)
{
    constexpr int step = 2 * ATT_WARPS;     // a pair of tiles for each warp
    return max(ATT_TPS, ((tiles + s_max - 1) / s_max + step - 1) / step * step);
}

template <int HD, bool ALONE>
__global__ void __launch_bounds__(32 * ATT_WARPS, att_ctas(HD)) k_kv4_attn(const Kv4Att a)
{
    constexpr int NB = HD / 32, TB = kv4_tile_bytes(HD), ST = ATT_STAGES, NT = 32 * ATT_WARPS;
    constexpr int IT = (8 * (HD / 4) + NT - 1) / NT;        // 4-value items of the output a thread joins
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t bars[ATT_WARPS][ST];
    __shared__ float sm_m[ATT_WARPS][8], sm_l[ATT_WARPS][8];
    // the queries' fragments and terms, made by one warp
    __shared__ __align__(16) uint4 sq[NB * 2 * 32];
    __shared__ float sks[32];
    float* so = reinterpret_cast<float*>(smem + ATT_WARPS * ST * 2 * TB);       // [warp][8][HD]
    pdl_trigger();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int G = a.heads / a.kv_heads, MG = (G + 7) / 8;
    const int kvh = blockIdx.y / MG, mg = blockIdx.y % MG, t = blockIdx.z, sp = blockIdx.x;
    const int nh = min(8, G - 8 * mg), head0 = kvh * G + 8 * mg;
    const int p = a.pos[t];
    const uint8_t* base = a.rows.base(t);
    const int state = kv4_row_state(base, p, a.capacity);
    if (state) {
        if (sp == 0)
            for (int i = threadIdx.x; i < nh * HD; i += NT)
                a.out[((int64_t)t * a.heads + head0) * HD + i] = state == 1 ? 0.f : NAN;
        return;
    }
    const Vis vis[1] = {visible(p, a.window, a.sinks)};
    const TileList tl = tile_list(vis[0].n, vis[0].first, vis[0].sink);
    const int range = att_range(tl.count, a.s_max), S = (tl.count + range - 1) / range;
    const bool alone = ALONE && S <= a.alone;
    if (sp >= (alone ? 1 : S)) return;
    const int i0 = sp * range, i1 = alone ? tl.count : min(tl.count, i0 + range);
    // step i of the warp: the pair of tiles at list item at(i) and the next (a range holds whole rounds of the warps' pairs)
    auto at = [&](int i) { return i0 + 2 * (i * ATT_WARPS + warp); };
    const int steps = max(0, (i1 - i0 - 2 * warp + 2 * ATT_WARPS - 1) / (2 * ATT_WARPS));
    uint8_t* ring = smem + warp * ST * 2 * TB;
    const uint8_t* src = base + (int64_t)kvh * TB;
    auto issue = [&](int i) {
        uint64_t* bar = &bars[warp][i % ST];
        const int x = at(i), two = x + 1 < i1;
        mbar_expect_tx(bar, two ? 2 * TB : TB);
        bulk_load(ring + i % ST * 2 * TB, src + (int64_t)tl.at(x) * a.kv_heads * TB, TB, bar);
        if (two) bulk_load(ring + i % ST * 2 * TB + TB, src + (int64_t)tl.at(x + 1) * a.kv_heads * TB, TB, bar);
    };
    if (lane == 0) {
        for (int s = 0; s < ST; ++s) mbar_init(&bars[warp][s], 1);
        fence_mbar_init();
        for (int s = 0; s < ST && s < steps; ++s) issue(s);
    }
    if (warp == 0) {
        uint4 qa[NB][2];
        float ks;
        load_query<HD>(g < nh ? a.q + ((int64_t)t * a.heads + head0 + g) * HD : nullptr, lane, a.scale * 1.4426950408889634f, qa, ks);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            sq[b * 64 + lane] = qa[b][0];
            sq[b * 64 + 32 + lane] = qa[b][1];
        }
        sks[lane] = ks;
    }
    __syncthreads();
    auto qf = [&](int, int b, int s) { return sq[b * 64 + s * 32 + lane]; };
    JoinState js[IT];
    int i = 0;
    bool ok = true;
    for (int r0 = i0; r0 < i1 && ok; r0 += range) {
        const int r1 = ALONE ? min(i1, r0 + range) : i1;
        AttState<HD, 1> st;
        st.init();
        for (; i < steps && (!ALONE || at(i) < r1); ++i) {
            ok = __all_sync(0xffffffffu, mbar_wait_bounded(&bars[warp][i % ST], (uint32_t)(i / ST & 1), a.err, 21));
            if (!ok) break;
            const int x = at(i);
            // (of an odd range's last step the second tile is not there: a position that no row sees)
            const int tile0[2] = {tl.at(x) * KV4_P, x + 1 < i1 ? tl.at(x + 1) * KV4_P : INT_MAX - KV4_P};
            const bool full = tile0[0] >= vis[0].first && tile0[1] < vis[0].n - KV4_P + 1;
            const float ks[1] = {sks[lane]};
            kv4_tiles<HD, 1, 2>(ring + i % ST * 2 * TB, lane, tile0, vis, full, qf, ks, st);
            __syncwarp();
            if (lane == 0 && i + ST < steps) issue(i + ST);
        }
        // the warps' sums of the range
        st.l[0] += __shfl_xor_sync(0xffffffffu, st.l[0], 1);
        st.l[0] += __shfl_xor_sync(0xffffffffu, st.l[0], 2);
        const float undo = 1.f / st.vs;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float4 v;
                v.x = st.sum(0, 4 * b, e) * undo;
                v.y = st.sum(0, 4 * b + 1, e) * undo;
                v.z = st.sum(0, 4 * b + 2, e) * undo;
                v.w = st.sum(0, 4 * b + 3, e) * undo;
                *reinterpret_cast<float4*>(so + (warp * 8 + g) * HD + 32 * b + 8 * c + 4 * e) = v;
            }
        if (c == 0) {
            sm_m[warp][g] = st.m[0];
            sm_l[warp][g] = st.l[0];
        }
        ok = __syncthreads_and(ok);         // (a wait that gave up ends the row for all warps)
#pragma unroll
        for (int k = 0; k < IT; ++k) {
            const int it = threadIdx.x + NT * k, h = it / (HD / 4), d = it % (HD / 4) * 4;
            if (h >= 8) break;
            float M = sm_m[0][h];
#pragma unroll
            for (int w = 1; w < ATT_WARPS; ++w) M = fmaxf(M, sm_m[w][h]);
            const float mu = M == -INFINITY ? 0.f : M;
            float L = 0.f;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < ATT_WARPS; ++w) {
                const float f = ex2(sm_m[w][h] - mu);
                const float4 x = *reinterpret_cast<const float4*>(so + (w * 8 + h) * HD + d);
                L = __fmaf_rn(f, sm_l[w][h], L);
                o.x = __fmaf_rn(f, x.x, o.x);
                o.y = __fmaf_rn(f, x.y, o.y);
                o.z = __fmaf_rn(f, x.z, o.z);
                o.w = __fmaf_rn(f, x.w, o.w);
            }
            js[k].add(M, L, o, r0 == i0);
        }
        if (!ALONE) break;
        if (r1 < i1) __syncthreads();       // (the next range's sums go to the same place)
    }
    // (after a wait that gave up, the warp's copies from step i on are still in flight; else none is)
    if (!ok && lane == 0)
        for (int x = i; x < min(steps, i + ST); ++x) mbar_drain(&bars[warp][x % ST], (uint32_t)(x / ST & 1));
#pragma unroll
    for (int k = 0; k < IT; ++k) {
        const int it = threadIdx.x + NT * k, h = it / (HD / 4), d = it % (HD / 4) * 4;
        if (h >= nh) continue;
        const int64_t th = (int64_t)t * a.heads + head0 + h;
        if (S == 1 || alone) {
            *reinterpret_cast<float4*>(a.out + th * HD + d) = js[k].out();
        } else {
            *reinterpret_cast<float4*>(a.part + (th * a.S + sp) * HD + d) = js[k].o;
            if (d == 0) reinterpret_cast<float2*>(a.ml)[th * a.S + sp] = make_float2(js[k].M, js[k].L);
        }
    }
    if (S == 1 || alone) return;
    if (!last_ticket(a.tickets + t * gridDim.y + blockIdx.y, S)) return;
    join_ranges<HD, NT>(a.ml, a.part, a.out, a.S, nh, S, so, RowMap{(int64_t)t * a.heads + head0, 0, 8, 8});
}

// Runs of R rows that read one cache (prompts): the (row, head) pairs of a run and KV head are queries 0 .. R G - 1; a CTA
// takes QB of them, each warp MT tiles of 8, and all warps share each tile of the cache (one ring of bulk copies), so
// a tile's codes are unpacked once for 8 MT queries. Only for head sizes that wl_kv4_mma.cu does not take (96 and 256).
// Measured: 500 rows behind 4000 positions, 32 heads on 8 of 96 dims 387 us, 16 on 8 of 256 456 us: bound by mma.sync's rate
// and the unpacking (32 rows of 8 heads of 128 dims, 5000 positions: 54 us so, 30 by wl_kv4_mma.cu).
template <int HD, int MT>
__global__ void __launch_bounds__(32 * RUN_WARPS, 2) k_kv4_attn_run(const Kv4Att a, int q_blocks)
{
    constexpr int NB = HD / 32, TB = kv4_tile_bytes(HD), ST = 4, QW = 8 * MT, QB = RUN_WARPS * QW;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t fullb[ST], emptyb[ST];
    __shared__ int rng[4];
    uint4* sq = reinterpret_cast<uint4*>(smem + ST * TB);       // [warp][MT][NB][2][32]
    pdl_trigger();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int G = a.heads / a.kv_heads, kvh = blockIdx.y;
    // the last queries (of a prompt: those that see most) first
    const int qb = q_blocks - 1 - (int)blockIdx.x / a.S, sp = blockIdx.x % a.S, run = blockIdx.z;
    const int nq = a.R * G, q0 = qb * QB;
    const uint8_t* base = a.rows.base(run * a.R);
    // the positions that the CTA's rows see together
    if (threadIdx.x == 0) {
        rng[0] = 0;
        rng[1] = INT_MAX;
        rng[2] = 0;
    }
    __syncthreads();
    {
        const int r0 = q0 / G, r1 = min(a.R - 1, (min(q0 + QB, nq) - 1) / G);
        for (int r = r0 + threadIdx.x; r <= r1; r += 32 * RUN_WARPS) {
            const int p = a.pos[run * a.R + r];
            if (kv4_row_state(base, p, a.capacity)) continue;
            const Vis v = visible(p, a.window, a.sinks);
            atomicMax(&rng[0], v.n);
            atomicMin(&rng[1], v.first);
            atomicMax(&rng[2], v.sink);
        }
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < ST; ++s) {
            mbar_init(&fullb[s], 1);
            mbar_init(&emptyb[s], RUN_WARPS);
        }
        fence_mbar_init();
    }
    __syncthreads();
    const TileList tl = rng[0] > 0 ? tile_list(rng[0], rng[1], rng[2]) : TileList{0, 0, 0};
    const int S = a.S;
    const int i0 = (int)((int64_t)tl.count * sp / S), i1 = (int)((int64_t)tl.count * (sp + 1) / S), nt = i1 - i0;
    const uint8_t* src = base + (int64_t)kvh * TB;
    auto issue = [&](int i) {
        uint64_t* bar = &fullb[i % ST];
        mbar_expect_tx(bar, TB);
        bulk_load(smem + i % ST * TB, src + (int64_t)tl.at(i0 + i) * a.kv_heads * TB, TB, bar);
    };
    if (threadIdx.x == 0)
        for (int s = 0; s < ST && s < nt; ++s) issue(s);
    Vis vis[MT];
    float ks[MT];
    int state[MT];
    int64_t th[MT];             // (row, head) of the lane's query, or -1
    int w_n = 0, w_min_n = INT_MAX, w_first = INT_MAX, w_max_first = 0, w_sink = 0;
    uint4* wq = sq + warp * MT * NB * 64;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int qi = q0 + warp * QW + 8 * i + g;
        th[i] = -1;
        state[i] = 1;
        vis[i] = Vis{0, 0, 0};
        if (qi < nq) {
            const int t = run * a.R + qi / G;
            th[i] = (int64_t)t * a.heads + kvh * G + qi % G;
            const int p = a.pos[t];
            state[i] = kv4_row_state(base, p, a.capacity);
            if (!state[i]) vis[i] = visible(p, a.window, a.sinks);
        }
        uint4 qa[NB][2];
        // (a padding row's query may hold anything: it enters as zeros, and its sums are zeros)
        load_query<HD>(!state[i] ? a.q + th[i] * HD : nullptr, lane, a.scale * 1.4426950408889634f, qa, ks[i]);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int s = 0; s < 2; ++s) wq[((i * NB + b) * 2 + s) * 32 + lane] = qa[b][s];
        if (vis[i].n > 0) {
            w_n = max(w_n, vis[i].n);
            w_min_n = min(w_min_n, vis[i].n);
            w_first = min(w_first, vis[i].first);
            w_max_first = max(w_max_first, vis[i].first);
            w_sink = max(w_sink, vis[i].sink);
        }
        else w_min_n = 0;
    }
    w_n = __reduce_max_sync(0xffffffffu, w_n);
    w_min_n = __reduce_min_sync(0xffffffffu, w_min_n);
    w_first = __reduce_min_sync(0xffffffffu, w_first);
    w_max_first = __reduce_max_sync(0xffffffffu, w_max_first);
    w_sink = __reduce_max_sync(0xffffffffu, w_sink);
    __syncwarp();
    AttState<HD, MT> st;
    st.init();
    auto qf = [&](int i, int b, int s) { return wq[((i * NB + b) * 2 + s) * 32 + lane]; };
    int i = 0;
    for (; i < nt; ++i) {
        if (!__all_sync(0xffffffffu, mbar_wait_bounded(&fullb[i % ST], (uint32_t)(i / ST & 1), a.err, 22))) break;
        const int tile0 = tl.at(i0 + i) * KV4_P;
        if (tile0 < w_n && (tile0 + KV4_P > w_first || tile0 < w_sink)) {
            const bool full = tile0 + KV4_P <= w_min_n && tile0 >= w_max_first;
            const int t0[1] = {tile0};
            kv4_tiles<HD, MT, 1>(smem + i % ST * TB, lane, t0, vis, full, qf, ks, st);
        }
        __syncwarp();
        bool ok = true;
        if (lane == 0) {
            asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&emptyb[i % ST])) : "memory");
            if (warp == 0 && i + ST < nt) {
                ok = mbar_wait_bounded(&emptyb[i % ST], (uint32_t)(i / ST & 1), a.err, 23);
                if (ok) issue(i + ST);
            }
        }
        if (!__all_sync(0xffffffffu, ok)) break;
    }
    // (after a wait that gave up, the copies from tile i on are still in flight; else none is)
    if (threadIdx.x == 0)
        for (int x = i; x < min(nt, i + ST); ++x) mbar_drain(&fullb[x % ST], (uint32_t)(x / ST & 1));
    const float undo = 1.f / st.vs;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        st.l[i] += __shfl_xor_sync(0xffffffffu, st.l[i], 1);
        st.l[i] += __shfl_xor_sync(0xffffffffu, st.l[i], 2);
        if (th[i] < 0) continue;
        const bool whole = S == 1;
        const float f = !whole ? undo : state[i] == 2 ? NAN : st.l[i] != 0.f ? undo / st.l[i] : 0.f;
        float* dst = whole ? a.out + th[i] * HD : a.part + (th[i] * S + sp) * HD;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float4 v;
                v.x = st.sum(i, 4 * b, e) * f;
                v.y = st.sum(i, 4 * b + 1, e) * f;
                v.z = st.sum(i, 4 * b + 2, e) * f;
                v.w = st.sum(i, 4 * b + 3, e) * f;
                *reinterpret_cast<float4*>(dst + 32 * b + 8 * c + 4 * e) = v;
            }
        if (!whole && c == 0) reinterpret_cast<float2*>(a.ml)[th[i] * S + sp] = make_float2(st.m[i], state[i] == 2 ? NAN : st.l[i]);
    }
    if (S == 1) return;
    if (!last_ticket(a.tickets + ((int64_t)run * a.kv_heads + kvh) * q_blocks + qb, S)) return;
    join_ranges<HD, 32 * RUN_WARPS>(a.ml, a.part, a.out, S, min(QB, nq - q0), S, reinterpret_cast<float*>(smem),
                                    RowMap{(int64_t)run * a.R * a.heads + kvh * G, q0, G, a.heads});
}

constexpr int64_t KV4_TICKETS = 1 << 18;    // tickets at the head of a workspace (zero between calls)

// Rows of a run up to which each is attended to by itself. 9 rows, 32 heads on 4, 4000 positions: 16 us so, 37 by tensor
// cores and 67 by k_kv4_attn_run; 12 rows of 500 positions: 10, 21 and 34; 16 rows of 3000: 28, 32 and 64. The rule looks at
// the rows alone, so it is wrong for few rows of many heads over a long cache (10 rows, 64 heads on 8, 20000 positions: 100,
// 65 and 161): there a rule on heads and room as well would gain a third.
constexpr int RUN_MIN_ROWS = 17;
constexpr int RUN_MAX_RANGES = 32;          // ranges a run may be cut into

// How a call is cut.
struct Kv4Plan {
    bool runs, mma, pairs;  // the rows' runs share their cache's tiles: on the tensor cores (k_kv4_attn_mma, in pairs of CTAs) or k_kv4_attn_run
    int S, s_max, alone, q_blocks, MT, MG;
    int64_t part_floats;
};

Kv4Plan kv4_plan(int T, int R, int heads, int kv_heads, int head_dim, int64_t capacity, int window, int sinks)
{
    Kv4Plan p{};
    const int G = heads / kv_heads;
    p.MG = (G + 7) / 8;
    int64_t tiles = (capacity + KV4_P - 1) / KV4_P;
    if (window > 0) tiles = std::min<int64_t>(tiles, ((int64_t)window + 15) / 16 + 1 + ((int64_t)sinks + 15) / 16);
    p.runs = R >= RUN_MIN_ROWS;
    // (32 and 64 rows of one query each, 5000 positions: 30 and 37 us by tensor cores, 54 and 75 by k_kv4_attn_run)
    p.mma = p.runs && (head_dim == 64 || head_dim == 128);
    p.MT = head_dim <= 128 ? 2 : 1;
    const int QB = p.mma ? 128 : RUN_WARPS * 8 * p.MT;
    p.q_blocks = (int)(((int64_t)R * G + QB - 1) / QB);
    p.pairs = p.mma && p.q_blocks > 1;
    if (p.pairs) p.q_blocks += p.q_blocks & 1;
    int64_t ctas;
    if (p.runs) {
        // as many ranges as end soonest: waves of CTAs over the SMs (two an SM, with CTAs of four warps), each of a range's
        // share of the tiles and 12 tiles' time to start and end (measured of k_kv4_attn_run: 8000 cycles against 5000 for 8 tiles)
        ctas = (int64_t)(T / R) * p.q_blocks * kv_heads;
        const int64_t slots = p.mma ? 148 : 2 * 148;
        double least = 1e30;
        for (int S = 1; S <= std::max<int64_t>(1, std::min<int64_t>(RUN_MAX_RANGES, tiles / 16)); ++S) {
            const double cost = (double)((ctas * S + slots - 1) / slots) * ((double)tiles / S + 12.0);
            if (cost < least) {
                least = cost;
                p.s_max = S;
            }
        }
        p.S = p.s_max;
    } else {
        // the most ranges of one row, from the shape alone (a row's bits must not depend on the others): one row's
        // CTAs fill the SMs two deep.
        ctas = (int64_t)T * kv_heads * p.MG;
        p.s_max = std::max(1, std::min(ATT_MAX_RANGES, 2 * 148 / (kv_heads * p.MG)));
        p.S = (int)std::max<int64_t>(1, std::min<int64_t>(p.s_max, (tiles + ATT_TPS - 1) / ATT_TPS));
        // enough rows for the SMs: short ones are walked by one CTA each (64 rows with a window of 1024: 49.7 us with a CTA a
        // range); a row of more than 8 ranges among them is still spread, so that the call does not wait for it. Beyond 64
        // rows every row is walked by one CTA a KV head, whatever its length, so that calls of any size need no partials: the
        // same ranges joined in the same order, so the same bits, but the call does wait for its longest row. (100 rows of 1000 to
        // 4000 positions, 32 heads on 8: 127 us so, 109 us with one range a row, which gave long rows other bits than alone.)
        p.alone = T > 64 || ctas > KV4_TICKETS ? INT_MAX : ctas >= 2 * 148 ? 8 : 0;
        if (p.alone >= p.S) p.S = 1;
    }
    if (p.runs && ctas > KV4_TICKETS) p.S = p.s_max = 1;
    p.part_floats = p.S > 1 ? (int64_t)T * heads * p.S * (head_dim + 2) : 0;
    return p;
}

template <int HD, bool ALONE> void attn_rows(const Kv4Att& a, const Kv4Plan& p, cudaStream_t s)
{
    constexpr int smem = ATT_WARPS * ATT_STAGES * 2 * kv4_tile_bytes(HD) + ATT_WARPS * 8 * HD * 4;
    static std::atomic<bool> done[64];
    ensure_smem_attr(k_kv4_attn<HD, ALONE>, smem, done);
    launch(k_kv4_attn<HD, ALONE>, dim3(p.S, a.kv_heads * p.MG, a.T), dim3(32 * ATT_WARPS), smem, s, a);
    note_launch();
}

template <int HD> void attn_rows(const Kv4Att& a, const Kv4Plan& p, cudaStream_t s)
{
    p.alone ? attn_rows<HD, true>(a, p, s) : attn_rows<HD, false>(a, p, s);
}

template <int HD> void attn_runs(const Kv4Att& a, const Kv4Plan& p, cudaStream_t s)
{
    constexpr int MT = HD <= 128 ? 2 : 1;
    // the ring and the queries' fragments; then the join's factors in their place
    constexpr int smem = 4 * kv4_tile_bytes(HD) + RUN_WARPS * MT * (HD / 32) * 2 * 512;
    static_assert(smem >= RUN_WARPS * 8 * MT * (3 * RUN_MAX_RANGES + 1) * 4, "the join's factors fit");
    static std::atomic<bool> done[64];
    ensure_smem_attr(k_kv4_attn_run<HD, MT>, smem, done);
    launch(k_kv4_attn_run<HD, MT>, dim3(p.q_blocks * p.S, a.kv_heads, a.T / a.R), dim3(32 * RUN_WARPS), smem, s, a, p.q_blocks);
    note_launch();
}

template <int HD>
void append_hd(const float* q, float* q_out, const float* k, const float* v, int T, int heads, int kv_heads, const float* table,
               int rope_dims, int neox, const Kv4Rows& rows, const int32_t* pos, int64_t capacity, cudaStream_t s)
{
    const int kv_blocks = (2 * kv_heads * (HD / 8) + 127) / 128;
    const int q_blocks = rope_dims > 0 || q_out != q ? (heads * (HD / 4) + 128 * APP_Q - 1) / (128 * APP_Q) : 0;
    const bool vec = rope_dims % 16 == 0 && (uintptr_t)table % 16 == 0;
    launch(vec ? k_kv4_append<HD, true> : k_kv4_append<HD, false>, dim3(kv_blocks + q_blocks, std::min(T, 65535)), dim3(128), 0, s, q, q_out,
           k, v, T, heads, kv_heads, table, rope_dims, neox, rows, pos, capacity, kv_blocks);
    note_launch();
}

template <int HD>
void read_hd(const Kv4Rows& rows, const int32_t* pos, int T, int kv_heads, int64_t capacity, void* k, void* v, cudaStream_t s)
{
    launch(k_kv4_read<HD>, dim3((2 * kv_heads * (HD / 8) + 127) / 128, std::min(T, 65535)), dim3(128), 0, s, rows, pos, T,
           kv_heads, capacity, (__half*)k, (__half*)v);
    note_launch();
}

}  // namespace

bool kv4_supported(int heads, int kv_heads, int head_dim)
{
    return heads > 0 && kv_heads > 0 && heads % kv_heads == 0 &&
           (head_dim == 64 || head_dim == 96 || head_dim == 128 || head_dim == 256);
}

int64_t kv4_bytes(int kv_heads, int head_dim, int64_t positions)
{
    return (positions + KV4_P - 1) / KV4_P * kv_heads * kv4_tile_bytes(head_dim);
}

int64_t kv4_workspace_bytes(int T, int R, int heads, int kv_heads, int head_dim, int64_t capacity, int window, int sinks)
{
    return KV4_TICKETS * 4 + 4 * kv4_plan(T, R, heads, kv_heads, head_dim, capacity, window, sinks).part_floats;
}

int64_t kv4_workspace_max(int above, int T, int heads, int kv_heads, int head_dim, int64_t capacity, int window, int sinks)
{
    // (every length: the ranges of neither kind fall steadily with it)
    int64_t most = 0;
    for (int t = above + 1; t <= T; ++t) {
        if (t <= 64) most = std::max(most, kv4_workspace_bytes(t, 1, heads, kv_heads, head_dim, capacity, window, sinks));
        most = std::max(most, kv4_workspace_bytes(t, t, heads, kv_heads, head_dim, capacity, window, sinks));
    }
    return most;
}

size_t kv4_ticket_bytes() { return (size_t)KV4_TICKETS * 4; }

void kv4_append(const float* q, float* q_out, const float* k, const float* v, int T, int heads, int kv_heads, int head_dim,
                const float* table, int rope_dims, int neox, const Kv4Cache& cache, const int32_t* pos, int64_t capacity,
                cudaStream_t s)
{
    if (T <= 0) return;
    const Kv4Rows r{(const uint8_t*)cache.rows, cache.pitch, cache.layer};
    switch (head_dim) {
    case 64: append_hd<64>(q, q_out, k, v, T, heads, kv_heads, table, rope_dims, neox, r, pos, capacity, s); break;
    case 96: append_hd<96>(q, q_out, k, v, T, heads, kv_heads, table, rope_dims, neox, r, pos, capacity, s); break;
    case 128: append_hd<128>(q, q_out, k, v, T, heads, kv_heads, table, rope_dims, neox, r, pos, capacity, s); break;
    default: append_hd<256>(q, q_out, k, v, T, heads, kv_heads, table, rope_dims, neox, r, pos, capacity, s); break;
    }
}

void kv4_read(const Kv4Cache& cache, const int32_t* pos, int T, int kv_heads, int head_dim, int64_t capacity, void* k, void* v,
              cudaStream_t s)
{
    if (T <= 0) return;
    const Kv4Rows r{(const uint8_t*)cache.rows, cache.pitch, cache.layer};
    switch (head_dim) {
    case 64: read_hd<64>(r, pos, T, kv_heads, capacity, k, v, s); break;
    case 96: read_hd<96>(r, pos, T, kv_heads, capacity, k, v, s); break;
    case 128: read_hd<128>(r, pos, T, kv_heads, capacity, k, v, s); break;
    default: read_hd<256>(r, pos, T, kv_heads, capacity, k, v, s); break;
    }
}

void kv4_attention(const float* q, int T, int R, int heads, int kv_heads, int head_dim, float scale, const Kv4Cache& cache,
                   const int32_t* pos, int64_t capacity, int window, int sinks, float* out, void* ws, int* err, cudaStream_t s)
{
    if (T <= 0) return;
    const Kv4Plan p = kv4_plan(T, R, heads, kv_heads, head_dim, capacity, window, sinks);
    // (a launch takes 65535 rows or runs; calls of more have one range a row and no partials)
    const int unit = p.runs ? R : 1;
    for (int64_t t0 = 0; t0 < T; t0 += (int64_t)65535 * unit) {
        Kv4Att a{};
        a.q = q + t0 * heads * head_dim;
        a.out = out + t0 * heads * head_dim;
        a.rows = Kv4Rows{(const uint8_t*)cache.rows + t0 * cache.pitch, cache.pitch, cache.layer};
        a.pos = pos + t0;
        a.T = (int)std::min<int64_t>(T - t0, (int64_t)65535 * unit);
        a.capacity = capacity; a.R = R; a.heads = heads; a.kv_heads = kv_heads; a.S = p.S; a.s_max = p.s_max; a.alone = p.alone;
        a.scale = scale; a.window = window; a.sinks = sinks;
        a.tickets = (int*)ws;
        a.part = (float*)((uint8_t*)ws + KV4_TICKETS * 4);
        a.ml = a.part + (int64_t)T * heads * p.S * head_dim;
        a.err = err;
        if (p.mma) kv4_attention_mma(a, head_dim, p.q_blocks, p.pairs, s);
        else switch (head_dim) {
        case 64: attn_rows<64>(a, p, s); break;
        case 96: p.runs ? attn_runs<96>(a, p, s) : attn_rows<96>(a, p, s); break;
        case 128: attn_rows<128>(a, p, s); break;
        default: p.runs ? attn_runs<256>(a, p, s) : attn_rows<256>(a, p, s); break;
        }
    }
}

}  // namespace k
}  // namespace wl
