// Selective state space scan along the rows of every region of a map: S states per channel that decay and take in the rows,
//
//   d = softplus(dt + bias) (or dt),  h[t] = exp(d A) h[t-1] + d x B[t],  y = C[t] . h[t] + D x,  y *= g sigmoid(g)
//
// with A (S, channels) per channel, B and C per row and group of channels. Backward, with e = dy g sigmoid(g) and the gradient g[t] of h[t]
// running from the last row to the first:
//
//   g[t] = C e + a[t+1] g[t+1],  dx = d (B . g) + D e,  dd = x (B . g) + sum_s g a h[t-1] A,  dA = sum_t g a h[t-1] d,
//   dB = sum over the group's channels of g d x,  dC = the same of e h,  dD = sum_t e x,  ddt = dd sigmoid(dt + bias),  dbias = sum_t ddt
//
// A lane is a channel: B and C are then the same for a whole wave whose channels are of one group, and come as scalar operands. Rows are
// taken 16 at a time (their x, d, y in registers) and states four at a time (in registers for the 16 rows, in LDS between), so that
// any number of states uses the same code. States are float32 (double for double rows).
#include <type_traits>
#include "rows_common.h"

namespace dbk {

constexpr unsigned SCAN_CHUNK = 16;              // rows taken together, and between two kept states
constexpr float LOG2E = 1.4426950408889634f;

struct scan_shape {
    unsigned N, D, S, G, gs, nregion;            // rows, channels, states, groups, channels per group, regions
    unsigned tpg, softplus;                      // waves' tiles per group (64 lanes per group), or 0: several groups per wave
    size_t ldx, lddt, ldb, ldc, ldg, ldy;
};

// The channel of a lane: LG = 64 lanes for the channels of one group (tpg tiles of 64), or LG lanes for each of 64 / LG groups.
struct scan_lane { unsigned group, ch; bool active; };
template <int LG> __device__ __forceinline__ scan_lane lane_channel(const scan_shape& p, unsigned tile, unsigned lane)
{
    scan_lane l;
    unsigned in;
    if (LG == 64) {
        l.group = tile / p.tpg;
        in = (tile - l.group * p.tpg) * 64u + lane;
        l.active = in < p.gs;
    } else {
        l.group = tile * (64u / LG) + lane / LG;
        in = lane % LG;
        l.active = l.group < p.G && in < p.gs;
        l.group = min(l.group, p.G - 1u);
    }
    l.ch = l.group * p.gs + min(in, p.gs - 1u);  // (a lane without a channel follows its group's last one and stores nothing)
    return l;
}

// four neighbouring weights of a row, those from `left` on zero; with UNIFORM the address is the same in all lanes and the loads are scalar
template <typename A, bool UNIFORM, bool FULL> __device__ __forceinline__ void load4(A (&v)[4], const A* p, unsigned left)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (UNIFORM) {
            typedef const __attribute__((address_space(4))) A* uniform_ptr;
            v[i] = FULL || i < (int)left ? ((uniform_ptr)(uintptr_t)p)[i] : A(0);
        } else
            v[i] = FULL || i < (int)left ? p[i] : A(0);
    }
}

__device__ __forceinline__ float fma_a(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ double fma_a(double a, double b, double c) { return fma(a, b, c); }

template <typename A> __device__ __forceinline__ A step_of(const scan_shape& p, A raw, A& slope)
{
    if (p.softplus) return softplus_of(raw, slope);
    slope = A(1);
    return raw;
}

template <typename A> struct quad { A v[4]; } __attribute__((aligned(16)));

// Forward over rows [from, to) of a region. h: the wave's states in LDS, [state / 4][lane] quads, holding those before row `from`.
// kept: null, or where the states before rows from + 16, from + 32, ... are written (one (S, D) block each).
template <typename T, int LG, bool WHOLE>
__device__ __forceinline__ void scan_chunk(const scan_shape& p, const scan_lane& l, unsigned lane, unsigned nrow, size_t row0, const T* X, const T* dt, const T* gate,
                                           const typename acc_of<T>::type* B, const typename acc_of<T>::type* C, typename acc_of<T>::type skip,
                                           typename acc_of<T>::type bias, quad<typename acc_of<T>::type>* h, const quad<typename acc_of<T>::type>* a2, T* Y)
{
    typedef typename acc_of<T>::type A;
    constexpr int R = SCAN_CHUNK;
    A d[R], in[R], y[R];
    T gt[R];
    const T *xr = X + row0 * p.ldx, *dr = dt + row0 * p.lddt;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (!WHOLE && i >= (int)nrow) break;
        const A x = (A)xr[(size_t)i * p.ldx + l.ch];
        A slope;
        d[i] = step_of(p, (A)dr[(size_t)i * p.lddt + l.ch] + bias, slope);
        in[i] = d[i] * x;
        y[i] = skip * x;
        if (gate) gt[i] = gate[(row0 + i) * p.ldg + l.ch];
    }
    auto states = [&](auto full, unsigned q) {
        constexpr bool FULL = decltype(full)::value;
        const quad<A> k = a2[q * 64u + lane];
        quad<A> s = h[q * 64u + lane];
        const A *br = B + row0 * p.ldb + (size_t)l.group * p.S + 4u * q, *cr = C + row0 * p.ldc + (size_t)l.group * p.S + 4u * q;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (!WHOLE && i >= (int)nrow) break;
            A b[4], c[4];
            load4<A, LG == 64, FULL>(b, br + (size_t)i * p.ldb, p.S - 4u * q);
            load4<A, LG == 64, FULL>(c, cr + (size_t)i * p.ldc, p.S - 4u * q);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s.v[j] = fma_a(exp2_fast(d[i] * k.v[j]), s.v[j], in[i] * b[j]);
                y[i] = fma_a(c[j], s.v[j], y[i]);
            }
        }
        h[q * 64u + lane] = s;
    };
    for (unsigned q = 0; 4u * q < p.S; ++q) {
        if (4u * q + 4u <= p.S) states(std::true_type(), q);
        else states(std::false_type(), q);
    }
    if (!l.active) return;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (!WHOLE && i >= (int)nrow) break;
        if (gate) { const A g = (A)gt[i]; y[i] *= g * sigmoid_of(g); }
        Y[(row0 + i) * p.ldy + l.ch] = (T)y[i];
    }
}

template <typename A> __device__ __forceinline__ void states_to(const scan_shape& p, const scan_lane& l, unsigned lane, const quad<A>* h, A* to)
{
    if (!l.active) return;
    for (unsigned q = 0; 4u * q < p.S; ++q) {
        const quad<A> s = h[q * 64u + lane];
#pragma unroll
        for (int j = 0; j < 4; ++j) if (4u * q + j < p.S) to[(size_t)(4u * q + j) * p.D + l.ch] = s.v[j];
    }
}
// zeros where there is nothing to read
template <typename A> __device__ __forceinline__ void states_from(const scan_shape& p, const scan_lane& l, unsigned lane, quad<A>* h, const A* from, A scale)
{
    for (unsigned q = 0; 4u * q < p.S; ++q) {
        quad<A> s;
#pragma unroll
        for (int j = 0; j < 4; ++j) s.v[j] = from && 4u * q + j < p.S ? from[(size_t)(4u * q + j) * p.D + l.ch] * scale : A(0);
        h[q * 64u + lane] = s;
    }
}

template <typename A> __device__ __forceinline__ A* kept_at(const scan_shape& p, A* keep, unsigned start, unsigned chunk)
{
    return keep + ((size_t)start / SCAN_CHUNK + chunk) * p.S * p.D;
}

// A wave per region and tile of channels.
template <typename T, int LG>
__global__ __launch_bounds__(64) void k_scan_fprop(scan_shape p, const uint32_t* __restrict__ regions, const T* __restrict__ X, const T* __restrict__ dt,
                                                   const typename acc_of<T>::type* __restrict__ A_, const typename acc_of<T>::type* __restrict__ B,
                                                   const typename acc_of<T>::type* __restrict__ C, const typename acc_of<T>::type* __restrict__ skip,
                                                   const T* __restrict__ gate, const typename acc_of<T>::type* __restrict__ bias,
                                                   const typename acc_of<T>::type* __restrict__ state, T* __restrict__ Y,
                                                   typename acc_of<T>::type* __restrict__ last, typename acc_of<T>::type* __restrict__ keep)
{
    typedef typename acc_of<T>::type A;
    extern __shared__ char lds_raw[];
    const unsigned lane = threadIdx.x, quads = (p.S + 3u) / 4u, r = blockIdx.x;
    quad<A>*h = (quad<A>*)lds_raw, *a2 = h + quads * 64u;
    const scan_lane l = lane_channel<LG>(p, blockIdx.y, lane);
    const row_range g = region_rows(regions, r, p.N);
    states_from(p, l, lane, a2, A_, A(1.4426950408889634));
    states_from(p, l, lane, h, state ? state + (size_t)r * p.S * p.D : (const A*)nullptr, A(1));
    const A sk = skip ? skip[l.ch] : A(0), bi = bias ? bias[l.ch] : A(0);
    unsigned chunk = 0;
    for (size_t row = g.start; row < g.end; row += SCAN_CHUNK, ++chunk) {
        const unsigned left = g.end - (unsigned)row;
        if (keep && chunk) states_to(p, l, lane, h, kept_at(p, keep, g.start, chunk));
        if (left >= SCAN_CHUNK) scan_chunk<T, LG, true>(p, l, lane, SCAN_CHUNK, row, X, dt, gate, B, C, sk, bi, h, a2, Y);
        else scan_chunk<T, LG, false>(p, l, lane, left, row, X, dt, gate, B, C, sk, bi, h, a2, Y);
    }
    if (last) states_to(p, l, lane, h, last + (size_t)r * p.S * p.D);
}

// ------------------------------------------------------------------------------------------------ sums over lanes
// Two values per lane become one: lanes with bit BIT of their number clear get the sum of a over the pair, the others that of b.
template <int CTRL> __device__ __forceinline__ float dpp_of(float x)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
template <int BIT> __device__ __forceinline__ float join(float a, float b, unsigned lane)
{
    if constexpr (BIT == 5) {                    // the upper half of a for the lower half of b: each lane then holds both terms of its sum
        const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
        return __uint_as_float(s[0]) + __uint_as_float(s[1]);
    } else if constexpr (BIT == 4) {
        const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
        return __uint_as_float(s[0]) + __uint_as_float(s[1]);
    } else {
        // partners: 8 lanes on in the row of 16; mirrored in the half row (which flips the two bits below too: the next two
        // steps meet the rest all the same); 2 and 1 lanes on in the quad
        constexpr int CTRL = BIT == 3 ? 0x128 : BIT == 2 ? 0x141 : BIT == 1 ? 0x4E : 0xB1;
        const bool up = (lane >> BIT) & 1u;
        return (up ? b : a) + dpp_of<CTRL>(up ? a : b);
    }
}
template <int BIT> __device__ __forceinline__ double join(double a, double b, unsigned lane)
{
    constexpr int MASK = BIT == 2 ? 7 : 1 << BIT;
    const bool up = (lane >> BIT) & 1u;
    return (up ? b : a) + __shfl_xor(up ? a : b, MASK);
}

struct scan_bshape { size_t lddy, lddx, ldddt, lddg, lddb, lddc; };

// Where a wave's sums of dB and dC go: the gradient itself where the wave holds the whole group, or its tile's share.
template <typename A> struct scan_out { A *dB, *dC; size_t ldb, ldc; };

// Backward over one chunk: the states are formed again from the one kept before it, then the rows are taken from the last to the first.
// lds: ag = the gradient that the rows behind send to the chunk's last state, da = dA so far, both [state / 4][lane]; st: two values per
// row and lane that are needed again at the end (the slope of the step; dY times the gate's derivative).
template <typename T, int LG, bool WHOLE>
__device__ __forceinline__ void scan_chunk_bprop(const scan_shape& p, const scan_bshape& bp, const scan_lane& l, unsigned lane, unsigned nrow, size_t row0, const T* X,
                                                 const T* dt, const T* gate, const T* dY, const typename acc_of<T>::type* B, const typename acc_of<T>::type* C,
                                                 typename acc_of<T>::type skip, typename acc_of<T>::type bias, const typename acc_of<T>::type* before,
                                                 const quad<typename acc_of<T>::type>* a2, quad<typename acc_of<T>::type>* ag, quad<typename acc_of<T>::type>* da,
                                                 typename acc_of<T>::type* st, T* dX, T* ddt, T* dgate, scan_out<typename acc_of<T>::type> out,
                                                 typename acc_of<T>::type& dskip, typename acc_of<T>::type& dbias)
{
    typedef typename acc_of<T>::type A;
    constexpr int R = SCAN_CHUNK;
    A x[R], d[R], e[R], sB[R], sA[R], y[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        x[i] = d[i] = e[i] = sB[i] = sA[i] = y[i] = A(0);
        if (!WHOLE && i >= (int)nrow) continue;
        x[i] = (A)X[(row0 + i) * p.ldx + l.ch];
        A slope;
        d[i] = step_of(p, (A)dt[(row0 + i) * p.lddt + l.ch] + bias, slope);
        e[i] = l.active ? (A)dY[(row0 + i) * bp.lddy + l.ch] : A(0);
        st[i * 64u + lane] = slope;
        if (gate) {
            const A g = (A)gate[(row0 + i) * p.ldg + l.ch], s = sigmoid_of(g);
            st[(R + i) * 64u + lane] = e[i] * s * fma_a(g, A(1) - s, A(1));
            e[i] *= g * s;
        }
    }
    auto states = [&](auto full, unsigned q) {
        constexpr bool FULL = decltype(full)::value;
        const unsigned left = p.S - 4u * q;
        const quad<A> k = a2[q * 64u + lane];
        const A *br = B + row0 * p.ldb + (size_t)l.group * p.S + 4u * q, *cr = C + row0 * p.ldc + (size_t)l.group * p.S + 4u * q;
        A h[R + 1][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) h[0][j] = before && (FULL || j < (int)left) ? before[(size_t)(4u * q + j) * p.D + l.ch] : A(0);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (!WHOLE && i >= (int)nrow) break;
            A b[4];
            load4<A, LG == 64, FULL>(b, br + (size_t)i * p.ldb, left);
            const A in = d[i] * x[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) h[i + 1][j] = fma_a(exp2_fast(d[i] * k.v[j]), h[i][j], in * b[j]);
        }
        quad<A> g = ag[q * 64u + lane], sum = da[q * 64u + lane];
        A rows[R];
#pragma unroll
        for (int i = R - 1; i >= 0; --i) {
            rows[i] = A(0);
            if (!WHOLE && i >= (int)nrow) continue;
            A b[4], c[4], v[8];
            load4<A, LG == 64, FULL>(b, br + (size_t)i * p.ldb, left);
            load4<A, LG == 64, FULL>(c, cr + (size_t)i * p.ldc, left);
            const A in = d[i] * x[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const A a = exp2_fast(d[i] * k.v[j]), now = fma_a(c[j], e[i], g.v[j]), w = now * (a * h[i][j]);
                if (gate) y[i] = fma_a(c[j], h[i + 1][j], y[i]);
                v[j] = now * in;
                v[4 + j] = e[i] * h[i + 1][j];
                sB[i] = fma_a(b[j], now, sB[i]);
                sA[i] = fma_a(w, k.v[j], sA[i]);
                sum.v[j] = fma_a(w, d[i], sum.v[j]);
                g.v[j] = a * now;
            }
            // eight values per row over three bits of the lane's number: one is left
            constexpr int TOP = LG == 64 ? 5 : LG == 32 ? 4 : 3;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = join<TOP>(v[j], v[4 + j], lane);
            v[0] = join<TOP - 1>(v[0], v[2], lane);
            v[1] = join<TOP - 1>(v[1], v[3], lane);
            rows[i] = join<TOP - 2>(v[0], v[1], lane);
        }
        ag[q * 64u + lane] = g;
        da[q * 64u + lane] = sum;
        // and the rows over the bits that are left: lane -> (matrix, state, rows)
        unsigned kind, state;
        if constexpr (LG == 64) {
            kind = lane >> 5;
            state = ((lane >> 4) & 1u) * 2u + ((lane >> 3) & 1u);
#pragma unroll
            for (int i = 0; i < 8; ++i) rows[i] = join<2>(rows[i], rows[i + 8], lane);
#pragma unroll
            for (int i = 0; i < 4; ++i) rows[i] = join<1>(rows[i], rows[i + 4], lane);
#pragma unroll
            for (int i = 0; i < 2; ++i) rows[i] = join<0>(rows[i], rows[i + 2], lane);
        } else if constexpr (LG == 32) {
            kind = (lane >> 4) & 1u;
            state = ((lane >> 3) & 1u) * 2u + ((lane >> 2) & 1u);
#pragma unroll
            for (int i = 0; i < 8; ++i) rows[i] = join<1>(rows[i], rows[i + 8], lane);
#pragma unroll
            for (int i = 0; i < 4; ++i) rows[i] = join<0>(rows[i], rows[i + 4], lane);
        } else {
            kind = (lane >> 3) & 1u;
            state = ((lane >> 2) & 1u) * 2u + ((lane >> 1) & 1u);
#pragma unroll
            for (int i = 0; i < 8; ++i) rows[i] = join<0>(rows[i], rows[i + 8], lane);
        }
        constexpr int LEFT = LG == 64 ? 2 : LG == 32 ? 4 : 8;                  // rows that a lane now holds
        const unsigned base = LG == 64 ? (lane & 1u) * 2u + ((lane >> 1) & 1u) * 4u + ((lane >> 2) & 1u) * 8u
                            : LG == 32 ? (lane & 1u) * 4u + ((lane >> 1) & 1u) * 8u : (lane & 1u) * 8u;
        // (lanes of a group that does not exist carry zeros into it and their first lane says so)
        if ((FULL || state < left) && (LG == 64 || l.active || (lane % LG >= p.gs && (lane / LG) + blockIdx.y * (64u / LG) < p.G))) {
            A* o = kind ? out.dC : out.dB;
            const size_t ld = kind ? out.ldc : out.ldb;
#pragma unroll
            for (int i = 0; i < LEFT; ++i)
                if (WHOLE || base + i < nrow) o[(row0 + base + i) * ld + (size_t)l.group * p.S + 4u * q + state] = rows[i];
        }
    };
    for (unsigned q = 0; 4u * q < p.S; ++q) {
        if (4u * q + 4u <= p.S) states(std::true_type(), q);
        else states(std::false_type(), q);
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (!WHOLE && i >= (int)nrow) continue;
        const A dd = fma_a(x[i], sB[i], sA[i] * A(0.6931471805599453)) * st[i * 64u + lane];      // (k is A log2(e))
        dskip = fma_a(e[i], x[i], dskip);
        dbias += dd;
        if (!l.active) continue;
        dX[(row0 + i) * bp.lddx + l.ch] = (T)fma_a(d[i], sB[i], skip * e[i]);
        ddt[(row0 + i) * bp.ldddt + l.ch] = (T)dd;
        if (gate) dgate[(row0 + i) * bp.lddg + l.ch] = (T)(fma_a(skip, x[i], y[i]) * st[(R + i) * 64u + lane]);
    }
}

// A wave per tile of channels takes its share of the regions one after another, with dA in LDS, and leaves one block of sums:
// part[unit][S + 2][D].
template <typename T, int LG>
__global__ __launch_bounds__(64) void k_scan_bprop(scan_shape p, scan_bshape bp, const uint32_t* __restrict__ regions, const T* __restrict__ X, const T* __restrict__ dt,
                                                   const typename acc_of<T>::type* __restrict__ A_, const typename acc_of<T>::type* __restrict__ B,
                                                   const typename acc_of<T>::type* __restrict__ C, const typename acc_of<T>::type* __restrict__ skip,
                                                   const T* __restrict__ gate, const typename acc_of<T>::type* __restrict__ bias,
                                                   const typename acc_of<T>::type* __restrict__ keep, const T* __restrict__ dY, T* __restrict__ dX,
                                                   T* __restrict__ ddt, T* __restrict__ dgate, scan_out<typename acc_of<T>::type> out,
                                                   size_t tile_stride, typename acc_of<T>::type* __restrict__ part)
{
    typedef typename acc_of<T>::type A;
    extern __shared__ char lds_raw[];
    const unsigned lane = threadIdx.x, quads = (p.S + 3u) / 4u;
    quad<A>*a2 = (quad<A>*)lds_raw, *ag = a2 + quads * 64u, *da = ag + quads * 64u;
    A* st = (A*)(da + quads * 64u);
    const scan_lane l = lane_channel<LG>(p, blockIdx.y, lane);
    states_from(p, l, lane, a2, A_, A(1.4426950408889634));
    states_from(p, l, lane, da, (const A*)nullptr, A(1));
    const A sk = skip ? skip[l.ch] : A(0), bi = bias ? bias[l.ch] : A(0);
    A dskip = 0, dbias = 0;
    if (LG == 64) {                              // (shares of a group's tiles lie one behind another)
        const size_t o = (size_t)(blockIdx.y - l.group * p.tpg) * tile_stride;
        out.dB += o;
        out.dC += o;
    }
    for (unsigned r = blockIdx.x; r < p.nregion; r += gridDim.x) {
        const row_range g = region_rows(regions, r, p.N);
        if (g.start == g.end) continue;
        states_from(p, l, lane, ag, (const A*)nullptr, A(1));
        for (unsigned chunk = (g.end - g.start - 1u) / SCAN_CHUNK + 1u; chunk-- > 0;) {
            const size_t row = (size_t)g.start + (size_t)chunk * SCAN_CHUNK;
            const unsigned left = g.end - (unsigned)row;
            const A* before = chunk ? kept_at(p, keep, g.start, chunk) : (const A*)nullptr;
            if (left >= SCAN_CHUNK)
                scan_chunk_bprop<T, LG, true>(p, bp, l, lane, SCAN_CHUNK, row, X, dt, gate, dY, B, C, sk, bi, before, a2, ag, da, st, dX, ddt, dgate, out, dskip, dbias);
            else
                scan_chunk_bprop<T, LG, false>(p, bp, l, lane, left, row, X, dt, gate, dY, B, C, sk, bi, before, a2, ag, da, st, dX, ddt, dgate, out, dskip, dbias);
        }
    }
    A* o = part + (size_t)blockIdx.x * (p.S + 2u) * p.D;
    states_to(p, l, lane, da, o);
    if (l.active) {
        o[(size_t)p.S * p.D + l.ch] = dskip;
        o[(size_t)(p.S + 1u) * p.D + l.ch] = dbias;
    }
}

// dB and dC of a region's rows from the tiles' shares, in the tiles' order.
template <typename A>
__global__ __launch_bounds__(256) void k_scan_weights(const uint32_t* __restrict__ regions, unsigned N, unsigned tiles, size_t ncol, const A* __restrict__ share,
                                                      size_t tile_stride, A* __restrict__ dB, size_t lddb, A* __restrict__ dC, size_t lddc)
{
    const row_range g = region_rows(regions, blockIdx.x, N);
    const size_t n = (size_t)(g.end - g.start) * 2u * ncol;
    for (size_t i = threadIdx.x; i < n; i += 256u) {
        const size_t row = g.start + i / (2u * ncol), c = i % (2u * ncol);
        A s = 0;
        for (unsigned t = 0; t < tiles; ++t) s += share[t * tile_stride + row * 2u * ncol + c];
        if (c < ncol) dB[row * lddb + c] = s;
        else dC[row * lddc + c - ncol] = s;
    }
}

// One new row per sequence: four waves share a tile of 64 channels, a quarter of the states each.
template <typename T>
__global__ __launch_bounds__(256) void k_scan_step(scan_shape p, const T* __restrict__ X, const T* __restrict__ dt, const typename acc_of<T>::type* __restrict__ A_,
                                                   const typename acc_of<T>::type* __restrict__ B, const typename acc_of<T>::type* __restrict__ C,
                                                   const typename acc_of<T>::type* __restrict__ skip, const T* __restrict__ gate,
                                                   const typename acc_of<T>::type* __restrict__ bias, const typename acc_of<T>::type* state,
                                                   typename acc_of<T>::type* into, T* __restrict__ Y)
{
    typedef typename acc_of<T>::type A;
    __shared__ A sums[4][64];
    const unsigned lane = threadIdx.x & 63u, part = threadIdx.x >> 6, ch = blockIdx.y * 64u + lane;
    const size_t r = blockIdx.x;
    const bool active = ch < p.D;
    A y = 0, x = 0;
    if (active) {
        A slope;
        x = (A)X[r * p.ldx + ch];
        const A d = step_of(p, (A)dt[r * p.lddt + ch] + (bias ? bias[ch] : A(0)), slope), in = d * x;
        const unsigned group = ch / p.gs, per = (p.S + 3u) / 4u;
        const A *b = B + r * p.ldb + (size_t)group * p.S, *c = C + r * p.ldc + (size_t)group * p.S;
        const unsigned stop = min(p.S, (part + 1u) * per);
#pragma unroll 4
        for (unsigned s = part * per; s < stop; ++s) {
            const size_t at = (r * p.S + s) * p.D + ch;
            const A h = fma_a(exp2_fast(d * (A_[(size_t)s * p.D + ch] * A(1.4426950408889634))), state[at], in * b[s]);
            into[at] = h;
            y = fma_a(c[s], h, y);
        }
    }
    sums[part][lane] = y;
    __syncthreads();
    if (part || !active) return;
    y = (sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
    y = fma_a(skip ? skip[ch] : A(0), x, y);
    if (gate) { const A g = (A)gate[r * p.ldg + ch]; y *= g * sigmoid_of(g); }
    Y[r * p.ldy + ch] = (T)y;
}

namespace {

constexpr unsigned SCAN_STATES = 64;             // the most states per channel: their LDS is 48 KiB a wave in the backward pass (float)
constexpr size_t SCAN_UNITS = 8192;              // waves that add up dA, over all tiles of channels

struct scan_plan { int lanes; unsigned tpg, tiles, units; };

scan_plan plan_scan(size_t D, size_t G, size_t P)
{
    scan_plan p;
    const size_t gs = D / G;
    p.lanes = gs <= 16 ? 16 : gs <= 32 ? 32 : 64;
    p.tpg = p.lanes == 64 ? divup(gs, 64) : 0u;
    p.tiles = p.lanes == 64 ? (unsigned)(G * p.tpg) : divup(G, 64 / p.lanes);
    const size_t cap = SCAN_UNITS / p.tiles ? SCAN_UNITS / p.tiles : 1;
    p.units = (unsigned)(P < cap ? P : cap);
    return p;
}

scan_shape shape_of(const dbk_statescan_args& a)
{
    scan_shape s;
    s.N = (unsigned)a.N; s.D = (unsigned)a.D; s.S = (unsigned)a.S; s.G = (unsigned)a.G; s.gs = (unsigned)(a.D / a.G); s.nregion = (unsigned)a.nregion;
    s.tpg = 0; s.softplus = a.softplus != 0;
    s.ldx = a.ldx; s.lddt = a.lddt; s.ldb = a.ldb; s.ldc = a.ldc; s.ldg = a.ldgate; s.ldy = a.ldy;
    return s;
}

template <typename F> void with_lanes(int lanes, F f)
{
    if (lanes == 16) f(std::integral_constant<int, 16>());
    else if (lanes == 32) f(std::integral_constant<int, 32>());
    else f(std::integral_constant<int, 64>());
}

int check_scan(const dbk_statescan_args* a)
{
    DBK_CHECK(a, "ValueError: null argument block");
    DBK_ROW_DTYPE_OK(a->dtype);
    DBK_CHECK(a->S >= 1 && a->S <= SCAN_STATES, "NotImplementedError: 1 to %u states per channel, got %zu", SCAN_STATES, a->S);
    DBK_CHECK(a->G >= 1 && a->D % a->G == 0, "ValueError: the number of channels must be divisible by the number of groups");
    DBK_CHECK(a->N < (size_t(1) << 32) - 64 && a->D < (size_t(1) << 21) && a->nregion < (size_t(1) << 31), "ValueError: map too large (%zu rows, %zu channels, %zu regions)",
              a->N, a->D, a->nregion);
    DBK_CHECK(!a->D || a->A, "ValueError: null weights");
    DBK_CHECK(!a->N || !a->D || (a->X && a->dt && a->B && a->C), "ValueError: null matrix");
    DBK_CHECK(a->N <= 1 || (a->ldx >= a->D && a->lddt >= a->D && a->ldb >= a->G * a->S && a->ldc >= a->G * a->S && (!a->gate || a->ldgate >= a->D)),
              "ValueError: row strides must be at least the number of columns");
    return 0;
}

size_t share_bytes(const dbk_statescan_args& a, const scan_plan& p)
{
    return p.tpg > 1 ? (size_t)p.tpg * a.N * 2 * a.G * a.S * acc_size(a.dtype) : 0;
}

}  // namespace
}  // namespace dbk

using namespace dbk;

extern "C" {

int dbk_statescan_args_size(void) { return (int)sizeof(dbk_statescan_args); }

int dbk_statescan_workspace(const dbk_statescan_args* a, int backward, size_t* work_bytes)
{
    if (int rc = check_scan(a)) return rc;
    DBK_CHECK(work_bytes, "ValueError: null result");
    *work_bytes = 0;
    if (a->N && a->D && a->nregion && backward) {
        const scan_plan p = plan_scan(a->D, a->G, a->nregion);
        *work_bytes = share_bytes(*a, p) + (size_t)p.units * (a->S + 2) * a->D * acc_size(a->dtype);
    }
    clear_error();
    return 0;
}

int dbk_statescan(dbk_stream_t stream, const dbk_statescan_args* a, void* work, size_t work_bytes)
{
    (void)work; (void)work_bytes;
    if (int rc = check_scan(a)) return rc;
    DBK_CHECK(!a->nregion || a->regions, "ValueError: null regions");
    DBK_CHECK(!a->N || !a->D || a->Y, "ValueError: null matrix");
    DBK_CHECK(a->N <= 1 || a->ldy >= a->D, "ValueError: row strides must be at least the number of columns");
    DBK_CHECK(!a->keep || !a->state, "ValueError: states are kept for the backward pass of whole sequences, which starts from zeros: no initial state");
    if (!a->D || !a->nregion) { clear_error(); return 0; }
    const scan_plan p = plan_scan(a->D, a->G, a->nregion);
    scan_shape s = shape_of(*a);
    s.tpg = p.tpg;
    hipStream_t st = as_stream(stream);
    with_row_type(a->dtype, [&](auto t) {
        typedef decltype(t) T;
        typedef typename acc_of<T>::type A;
        with_lanes(p.lanes, [&](auto lanes) {
            const size_t lds = (a->S + 3) / 4 * 64 * 2 * sizeof(quad<A>);
            k_scan_fprop<T, lanes.value><<<dim3((unsigned)a->nregion, p.tiles), 64, lds, st>>>(
                s, a->regions, (const T*)a->X, (const T*)a->dt, (const A*)a->A, (const A*)a->B, (const A*)a->C, (const A*)a->skip, (const T*)a->gate, (const A*)a->dt_bias,
                (const A*)a->state, (T*)a->Y, (A*)a->last, (A*)a->keep);
        });
    });
    DBK_LAUNCH_OK();
}

int dbk_statescan_bprop(dbk_stream_t stream, const dbk_statescan_args* a, void* work, size_t work_bytes)
{
    if (int rc = check_scan(a)) return rc;
    DBK_CHECK(!a->nregion || a->regions, "ValueError: null regions");
    DBK_CHECK(!a->D || a->dA, "ValueError: null gradient");
    DBK_CHECK(!a->N || !a->D || (a->dY && a->dX && a->ddt && a->dB && a->dC && (!a->gate || a->dgate)), "ValueError: null gradient");
    DBK_CHECK(!a->N || !a->D || a->keep, "ValueError: the states that the forward pass kept are needed");
    DBK_CHECK(a->N <= 1 || (a->lddy >= a->D && a->lddx >= a->D && a->ldddt >= a->D && a->lddb >= a->G * a->S && a->lddc >= a->G * a->S && (!a->gate || a->lddgate >= a->D)),
              "ValueError: row strides must be at least the number of columns");
    if (!a->D) { clear_error(); return 0; }
    hipStream_t st = as_stream(stream);
    if (!a->nregion || !a->N) {
        sum_partials(st, a->dtype, nullptr, 0, a->S * a->D, a->dA, a->D, a->dskip, a->D, a->ddt_bias);       // (sums of no rows: zeros)
        DBK_LAUNCH_OK();
    }
    size_t need = 0;
    if (int rc = dbk_statescan_workspace(a, 1, &need)) return rc;
    DBK_CHECK(work && work_bytes >= need, "ValueError: the workspace has %zu bytes, %zu are needed", work_bytes, need);
    const scan_plan p = plan_scan(a->D, a->G, a->nregion);
    scan_shape s = shape_of(*a);
    s.tpg = p.tpg;
    const scan_bshape b = {a->lddy, a->lddx, a->ldddt, a->lddgate, a->lddb, a->lddc};
    const size_t shares = share_bytes(*a, p), ncol = a->G * a->S;
    void* part = (char*)work + shares;
    with_row_type(a->dtype, [&](auto t) {
        typedef decltype(t) T;
        typedef typename acc_of<T>::type A;
        scan_out<A> out = {(A*)a->dB, (A*)a->dC, a->lddb, a->lddc};
        size_t tile_stride = 0;
        if (shares) {                            // a tile's share: (N, dB | dC)
            out = {(A*)work, (A*)work + ncol, 2 * ncol, 2 * ncol};
            tile_stride = a->N * 2 * ncol;
        }
        with_lanes(p.lanes, [&](auto lanes) {
            const size_t lds = (a->S + 3) / 4 * 64 * 3 * sizeof(quad<A>) + 2 * SCAN_CHUNK * 64 * sizeof(A);
            k_scan_bprop<T, lanes.value><<<dim3(p.units, p.tiles), 64, lds, st>>>(
                s, b, a->regions, (const T*)a->X, (const T*)a->dt, (const A*)a->A, (const A*)a->B, (const A*)a->C, (const A*)a->skip, (const T*)a->gate, (const A*)a->dt_bias,
                (const A*)a->keep, (const T*)a->dY, (T*)a->dX, (T*)a->ddt, (T*)a->dgate, out, tile_stride, (A*)part);
        });
        if (shares)
            k_scan_weights<A><<<(unsigned)a->nregion, 256, 0, st>>>(a->regions, (unsigned)a->N, p.tpg, ncol, (const A*)work, tile_stride, (A*)a->dB, a->lddb, (A*)a->dC, a->lddc);
    });
    sum_partials(st, a->dtype, part, p.units, a->S * a->D, a->dA, a->D, a->dskip, a->D, a->ddt_bias);
    DBK_LAUNCH_OK();
}

int dbk_statescan_step(dbk_stream_t stream, const dbk_statescan_args* a)
{
    if (int rc = check_scan(a)) return rc;
    DBK_CHECK(!a->N || !a->D || (a->Y && a->state && a->last), "ValueError: null matrix or state");
    DBK_CHECK(a->N <= 1 || a->ldy >= a->D, "ValueError: row strides must be at least the number of columns");
    DBK_CHECK(a->N < (size_t(1) << 31), "ValueError: too many sequences (%zu)", a->N);
    if (!a->N || !a->D) { clear_error(); return 0; }
    const scan_shape s = shape_of(*a);
    hipStream_t st = as_stream(stream);
    with_row_type(a->dtype, [&](auto t) {
        typedef decltype(t) T;
        typedef typename acc_of<T>::type A;
        k_scan_step<T><<<dim3((unsigned)a->N, divup(a->D, 64)), 256, 0, st>>>(s, (const T*)a->X, (const T*)a->dt, (const A*)a->A, (const A*)a->B, (const A*)a->C,
                                                                             (const A*)a->skip, (const T*)a->gate, (const A*)a->dt_bias, (const A*)a->state, (A*)a->last, (T*)a->Y);
    });
    DBK_LAUNCH_OK();
}

}  // extern "C"
