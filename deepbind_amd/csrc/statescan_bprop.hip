// The scan's backward pass. Formulas and layout: statescan.h.
#include "statescan.h"

namespace dbk {

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

template <typename A> struct quad { A v[4]; } __attribute__((aligned(16)));

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

namespace {

constexpr size_t SCAN_UNITS = 8192;              // waves that add up dA, over all tiles of channels

scan_plan plan_bprop(const dbk_statescan_args& a) { return plan_scan(a.N, a.D, a.G, 1, a.N + 1); }
unsigned bprop_units(const dbk_statescan_args& a, const scan_plan& p)
{
    const size_t cap = SCAN_UNITS / p.tiles ? SCAN_UNITS / p.tiles : 1;
    return (unsigned)(a.nregion < cap ? a.nregion : cap);
}
inline size_t share_bytes(const dbk_statescan_args& a, const scan_plan& p)
{
    return p.tpg > 1 ? (size_t)p.tpg * a.N * 2 * a.G * a.S * acc_size(a.dtype) : 0;
}

}  // namespace

size_t bprop_work_bytes(const dbk_statescan_args& a)
{
    const scan_plan p = plan_bprop(a);
    return share_bytes(a, p) + (size_t)bprop_units(a, p) * (a.S + 2) * a.D * acc_size(a.dtype);
}

}  // namespace dbk

using namespace dbk;

extern "C" {

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
    const size_t need = bprop_work_bytes(*a);
    DBK_CHECK(work && work_bytes >= need, "ValueError: the workspace has %zu bytes, %zu are needed", work_bytes, need);
    const scan_plan p = plan_bprop(*a);
    const unsigned units = bprop_units(*a, p);
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
            k_scan_bprop<T, lanes.value><<<dim3(units, p.tiles), 64, lds, st>>>(
                s, b, a->regions, (const T*)a->X, (const T*)a->dt, (const A*)a->A, (const A*)a->B, (const A*)a->C, (const A*)a->skip, (const T*)a->gate, (const A*)a->dt_bias,
                (const A*)a->keep, (const T*)a->dY, (T*)a->dX, (T*)a->ddt, (T*)a->dgate, out, tile_stride, (A*)part);
        });
        if (shares)
            k_scan_weights<A><<<(unsigned)a->nregion, 256, 0, st>>>(a->regions, (unsigned)a->N, p.tpg, ncol, (const A*)work, tile_stride, (A*)a->dB, a->lddb, (A*)a->dC, a->lddc);
    });
    sum_partials(st, a->dtype, part, units, a->S * a->D, a->dA, a->D, a->dskip, a->D, a->ddt_bias);
    DBK_LAUNCH_OK();
}

}  // extern "C"
