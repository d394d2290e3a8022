// The scan's backward pass. Formulas and layout: statescan.h.
//
// 459 vector instructions per row and wave with 16 states, 332 of them the states' own (per state two 2^x, four products and sums to
// form it again, ten on the way back, four for the sums over lanes). Eight rows are taken together because 16 would not fit the registers.
// Measured: 14 576 rows of 1024 bfloat16 channels in two long regions 290 us (and 104 for
// what enters their segments), 47 678 rows of 24 models of 16 floats, without a gate, 463 us (40 more with the gated form). The first are 2840 clocks of a SIMD
// per row and wave, where the instructions alone come to some 1490 at the rates measured one by one: two waves per SIMD issue 58 % of their time, wait for
// memory and LDS 27 %, for their turn 15 %, and the chains of dependent sums over lanes and of 2^x are not filled by other rows' work.
#include "statescan.h"

namespace dbk {

// States go through the kernel by fours. What is left over of the last four follows the last state: the same decay, input and start, and shares of its C and
// of what is sent to it that add up to one exactly, so that all its gradients are shares too, and no 0 * inf arises where the state has none. Their sum
// is the state's: for dX, ddt and the gate it is formed with the sum over states anyway.
// The exponent of the share of state s, which exists or follows.
__device__ __forceinline__ int share_exp(unsigned S, unsigned s) { return s + 1u < S ? 0 : -(int)min(s + 2u - S, (0u - S) & 3u); }

template <typename A> __device__ __forceinline__ void states_to(const scan_shape& p, const scan_lane& l, unsigned lane, const quad<A>* h, A* to)
{
    if (!l.active) return;
    const unsigned at = opaque(l.ch * (unsigned)sizeof(A));
    for (unsigned q = 0; 4u * q < p.S; ++q) {
        quad<A> s = h[q * 64u + lane];
#pragma unroll
        for (int j = 3; j > 0; --j) if (4u * q + j >= p.S) s.v[j - 1] += s.v[j];
#pragma unroll
        for (int j = 0; j < 4; ++j) if (4u * q + j < p.S) lane_store(to + (size_t)(4u * q + j) * p.D, at, s.v[j]);
    }
}
// zeros where there is nothing to read
template <typename A> __device__ __forceinline__ void states_from(const scan_shape& p, const scan_lane& l, unsigned lane, quad<A>* h, const A* from)
{
    const unsigned at = opaque(l.ch * (unsigned)sizeof(A));
    for (unsigned q = 0; 4u * q < p.S; ++q) {
        quad<A> s;
#pragma unroll
        for (int j = 0; j < 4; ++j) s.v[j] = from ? ldexp_a(lane_load(from + (size_t)min(4u * q + j, p.S - 1u) * p.D, at), share_exp(p.S, 4u * q + j)) : A(0);
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

template <typename T> struct scan_rows_in {      // what the backward pass reads of a row
    typedef typename acc_of<T>::type A;
    const T *X, *dt, *gate, *dY;
    const A *B, *C, *keep;
    const uint32_t *regions, *marks;
};
template <typename T> struct scan_rows_out { T *dX, *ddt, *dgate; };

// What a chunk of nrow <= 8 rows needs from memory, fetched into registers while the chunk behind it is worked on: the rows of its channels, and
// its share of B and C, which then lie in LDS as [row][B, C][group of the wave][state], zeros behind the last row (in LDS rather
// than in scalar registers, for which a row's work is too short to hide the loads of the next row's). With more than 16 states
// the weights come when they are needed.
template <typename T, int LG, bool GATED> struct scan_raw {
    typedef typename acc_of<T>::type A;
    static constexpr int R = SCAN_CHUNK, GW = 64 / LG, WIDTH = 2 * GW * 16, NW = R * WIDTH / 64;
    T x[R], d[R], e[R], g[R];
    A w[NW];
    // (rows behind the chunk's last one repeat it)
    __device__ __forceinline__ void fetch(const scan_shape& p, const scan_bshape& bp, const scan_lane& l, unsigned lane, unsigned nrow, size_t row0, const scan_rows_in<T>& in)
    {
        const unsigned place = opaque(l.ch * (unsigned)sizeof(T));
        const T *xp = in.X + row0 * p.ldx, *dp = in.dt + row0 * p.lddt, *ep = in.dY + row0 * bp.lddy;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            x[i] = lane_load(xp, place);
            d[i] = lane_load(dp, place);
            e[i] = lane_load(ep, place);
            const bool more = i + 1 < (int)nrow;
            xp += more ? p.ldx : 0;
            dp += more ? p.lddt : 0;
            ep += more ? bp.lddy : 0;
        }
        if constexpr (GATED) {
            const T* gp = in.gate + row0 * p.ldg;
#pragma unroll
            for (int i = 0; i < R; ++i) {
                g[i] = lane_load(gp, place);
                gp += i + 1 < (int)nrow ? p.ldg : 0;
            }
        }
        if (p.S > 16u) return;
        const unsigned first = first_group<LG>(p, blockIdx.y);
#pragma unroll
        for (int n = 0; n < NW; ++n) {
            const unsigned at = lane % 64u + 64u * n, in_row = at % WIDTH, r = at / WIDTH, gr = in_row % (GW * 16) / 16, s = in_row % 16u;
            const bool c = in_row >= GW * 16;
            const A* from = (c ? in.C + row0 * p.ldc : in.B + row0 * p.ldb) + ((size_t)r * (c ? p.ldc : p.ldb) + (size_t)(first + gr) * p.S + min(s, p.S - 1u));
            w[n] = first + gr < p.G && r < nrow ? *from : A(0);
        }
    }
    __device__ __forceinline__ void put(const scan_shape& p, unsigned lane, unsigned nrow, size_t row0, const scan_rows_in<T>& in, A* bc) const
    {
        if (p.S <= 16u) {
#pragma unroll
            for (int n = 0; n < NW; ++n) bc[lane + 64 * n] = w[n];
            if (p.S % 4u) {
#pragma unroll
                for (int n = 0; n < NW; ++n) {
                    const unsigned at = lane + 64u * n;
                    if (at % WIDTH >= GW * 16) bc[at] = ldexp_a(w[n], share_exp(p.S, at % 16u));
                }
            }
        } else {
            const unsigned pad = (p.S + 3u) / 4u * 4u, width = 2u * GW * pad, first = first_group<LG>(p, blockIdx.y);
            for (unsigned i = lane; i < width; i += 64u) {
                const unsigned gr = i / pad % GW, s = i % pad;
                const bool c = i >= GW * pad, here = first + gr < p.G;
                const A* from = (c ? in.C + row0 * p.ldc : in.B + row0 * p.ldb) + (size_t)(first + gr) * p.S + min(s, p.S - 1u);
                const size_t ld = c ? p.ldc : p.ldb;
                const int share = c ? share_exp(p.S, s) : 0;
#pragma unroll
                for (unsigned r = 0; r < (unsigned)R; ++r) bc[r * width + i] = here && r < nrow ? ldexp_a(from[r * ld], share) : A(0);
            }
        }
        __builtin_amdgcn_wave_barrier();         // (one wave: LDS keeps its order)
    }
};
template <typename T> __device__ __forceinline__ unsigned weights_pad(unsigned S) { return S <= 16u ? 16u : (S + 3u) / 4u * 4u; }

// Backward over one chunk of nrow <= 8 rows: the states are formed again from the one kept before it, then the rows are taken from the last
// to the first; four states at a time, whose values at all rows are in registers, while those of the other states wait in LDS.
// ag: the gradient that the rows behind send to the chunk's last state, da: dA so far, both [state / 4][lane]; st: two values per
// row and lane that are needed again at the end (the slope of the step; dY times the gate's derivative); bc: the weights (scan_raw). raw: this
// chunk's values, and on return those of the one in front of it, which starts `ahead` rows earlier (0: there is none).
template <typename T, int LG, bool GATED>
__device__ __forceinline__ void scan_chunk_bprop(const scan_shape& p, const scan_bshape& bp, const scan_lane& l, unsigned lane, unsigned nrow, size_t row0,
                                                 const scan_rows_in<T>& in, const typename acc_of<T>::type* A_, typename acc_of<T>::type skip,
                                                 typename acc_of<T>::type bias, const typename acc_of<T>::type* before,
                                                 quad<typename acc_of<T>::type>* ag, quad<typename acc_of<T>::type>* da, typename acc_of<T>::type* st,
                                                 typename acc_of<T>::type* bc, scan_raw<T, LG, GATED>& raw, unsigned ahead, const scan_rows_out<T>& to,
                                                 scan_out<typename acc_of<T>::type> out, typename acc_of<T>::type& dskip, typename acc_of<T>::type& dbias)
{
    typedef typename acc_of<T>::type A;
    constexpr int R = SCAN_CHUNK;
    const unsigned place = opaque(l.ch * (unsigned)sizeof(T)), place_a = opaque(l.ch * (unsigned)sizeof(A));
    // what the next four states start from is fetched while these are worked on
    quad<A> kn, hn;
    auto fetch = [&](unsigned q) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const unsigned s = min(4u * q + j, p.S - 1u);
            kn.v[j] = lane_load(A_ + (size_t)s * p.D, place_a);
            hn.v[j] = before ? lane_load(before + (size_t)s * p.D, place_a) : A(0);
        }
    };
    fetch(0);
    A x[R], d[R], e[R], sB[R], sA[R], y[R];
    {
        raw.put(p, lane, nrow, row0, in, bc);
        if (p.softplus) {
#pragma unroll
            for (int i = 0; i < R; ++i) {
                A slope;
                d[i] = softplus_of((A)raw.d[i] + bias, slope);
                st[i * 64u + lane] = slope;
            }
        } else {
#pragma unroll
            for (int i = 0; i < R; ++i) {
                d[i] = (A)raw.d[i] + bias;
                st[i * 64u + lane] = A(1);
            }
        }
        // rows behind the last one, and lanes without a channel, whose sums go into their group's: no step, so nothing is taken in or sent
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const bool here = i < (int)nrow && l.active;
            A ee = (A)raw.e[i];
            if constexpr (GATED) {
                const A g = (A)raw.g[i], s = sigmoid_of(g);
                st[(R + i) * 64u + lane] = ee * s * fma_a(g, A(1) - s, A(1));
                ee *= g * s;
            }
            x[i] = here ? (A)raw.x[i] : A(0);
            d[i] = here ? d[i] : A(0);
            e[i] = here ? ee : A(0);
            sB[i] = sA[i] = A(0);
            if (GATED) y[i] = skip * x[i];
        }
    }
    if (ahead) raw.fetch(p, bp, l, lane, SCAN_CHUNK, row0 - ahead, in);
    const unsigned pad = weights_pad<T>(p.S), width = 2u * (64 / LG) * pad;
    const A* weights = bc + (lane / LG) * pad;
    for (unsigned q = 0; 4u * q < p.S; ++q) {
        const unsigned left = p.S - 4u * q;
        quad<A> k = kn;
        A h[R + 1][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            k.v[j] = l.active ? k.v[j] * A(1.4426950408889634) : A(0);
            h[0][j] = l.active ? hn.v[j] : A(0);
        }
        if (left > 4u) fetch(q + 1u);
        const A *b = weights + 4u * q, *c = b + (64 / LG) * pad;
        quad<A> bn = *(const quad<A>*)b;
        // A row's work stays together, its weights being fetched a row ahead: left to itself the compiler gathers many rows' weights and
        // spills them. Rows that do not exist are left out by fours.
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (i % 4 == 0 && i >= (int)nrow) break;
            const quad<A> bi = bn;
            if (i + 1 < R) bn = *(const quad<A>*)(b + (i + 1) * width);
            const A dx = d[i] * x[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) h[i + 1][j] = fma_a(exp2_fast(d[i] * k.v[j]), h[i][j], dx * bi.v[j]);
            __builtin_amdgcn_sched_barrier(0);
        }
        // (the decays, like the product of step and input, are formed again below: kept from the first time they would take 40 registers
        // more, and the compiler is told nothing about their factors any more so that it does not keep them)
#pragma unroll
        for (int j = 0; j < 4; ++j) k.v[j] = opaque(k.v[j]);
#pragma unroll
        for (int i = 0; i < R; ++i) x[i] = opaque(x[i]);
        quad<A> g = ag[q * 64u + lane], sum = da[q * 64u + lane];
        A rows[R];
#pragma unroll
        for (int i = R - 1; i >= 0; --i) {
            rows[i] = A(0);
            if (i >= (int)nrow) continue;
            const quad<A> bi = *(const quad<A>*)(b + i * width), ci = *(const quad<A>*)(c + i * width);
            const A dx = d[i] * x[i];
            A v[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const A a = exp2_fast(d[i] * k.v[j]), now = fma_a(ci.v[j], e[i], g.v[j]), w = now * (a * h[i][j]);
                if (GATED) y[i] = fma_a(ci.v[j], h[i + 1][j], y[i]);
                v[j] = now * dx;
                v[4 + j] = e[i] * h[i + 1][j];
                sB[i] = fma_a(bi.v[j], now, sB[i]);
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
            // and the rows over the bits that are left, the first of them as soon as both are there
            if (i < R / 2) rows[i] = join<TOP - 3>(rows[i], rows[i + R / 2], lane);
            __builtin_amdgcn_sched_barrier(0);
        }
        ag[q * 64u + lane] = g;
        da[q * 64u + lane] = sum;
        // lane -> (matrix, state, rows)
        unsigned kind, state;
        if constexpr (LG == 64) {
            kind = lane >> 5;
            state = ((lane >> 4) & 1u) * 2u + ((lane >> 3) & 1u);
            rows[0] = join<1>(rows[0], rows[2], lane);
            rows[1] = join<1>(rows[1], rows[3], lane);
            rows[0] = join<0>(rows[0], rows[1], lane);
        } else if constexpr (LG == 32) {
            kind = (lane >> 4) & 1u;
            state = ((lane >> 3) & 1u) * 2u + ((lane >> 2) & 1u);
            rows[0] = join<0>(rows[0], rows[2], lane);
            rows[1] = join<0>(rows[1], rows[3], lane);
        } else {
            kind = (lane >> 3) & 1u;
            state = ((lane >> 2) & 1u) * 2u + ((lane >> 1) & 1u);
        }
        constexpr int LEFT = LG == 64 ? 1 : LG == 32 ? 2 : 4;                  // rows that a lane now holds
        const unsigned base = LG == 64 ? (lane & 1u) + ((lane >> 1) & 1u) * 2u + ((lane >> 2) & 1u) * 4u
                            : LG == 32 ? (lane & 1u) * 2u + ((lane >> 1) & 1u) * 4u : (lane & 1u) * 4u;
        if (left < 4u) {                         // (the last state's dB is in shares)
            constexpr int BIT1 = LG == 64 ? 16 : LG == 32 ? 8 : 4;
#pragma unroll
            for (int i = 0; i < LEFT; ++i) {
                A all = state + 1u >= left ? rows[i] : A(0);
                all += __shfl_xor(all, BIT1);
                all += __shfl_xor(all, BIT1 / 2);
                rows[i] = kind == 0u && state + 1u == left ? all : rows[i];
            }
        }
        // (lanes of a group that does not exist carry zeros into it and their first lane says so)
        if (state < left && (LG == 64 || l.active || (lane % LG >= p.gs && (lane / LG) + blockIdx.y * (64u / LG) < p.G))) {
            A* o = kind ? out.dC : out.dB;
            const size_t ld = kind ? out.ldc : out.ldb;
#pragma unroll
            for (int i = 0; i < LEFT; ++i)
                if (base + i < nrow) o[(row0 + base + i) * ld + (size_t)l.group * p.S + 4u * q + state] = rows[i];
        }
    }
    T *xp = to.dX + row0 * bp.lddx, *dp = to.ddt + row0 * bp.ldddt, *gp = to.dgate + row0 * bp.lddg;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (i >= (int)nrow) break;
        const A dd = fma_a(x[i], sB[i], sA[i] * A(0.6931471805599453)) * st[i * 64u + lane];      // (k is A log2(e))
        dskip = fma_a(e[i], x[i], dskip);
        dbias += dd;
        if (l.active) {
            lane_store(xp, place, (T)fma_a(d[i], sB[i], skip * e[i]));
            lane_store(dp, place, (T)dd);
            if constexpr (GATED) lane_store(gp, place, (T)(y[i] * st[(R + i) * 64u + lane]));
        }
        xp += bp.lddx;
        dp += bp.ldddt;
        gp += bp.lddg;
    }
}

// A wave's place in LDS and what it adds up over all its rows.
template <typename T, int LG, bool GATED> struct scan_wave {
    typedef typename acc_of<T>::type A;
    unsigned lane;
    scan_lane l;
    quad<A> *ag, *da;
    A *st, *bc, sk, bi, dskip, dbias;
    const A* A_;
    __device__ __forceinline__ scan_wave(const scan_shape& p, char* lds, const A* decay, const A* skip, const A* bias)
    {
        const unsigned quads = (p.S + 3u) / 4u;
        lane = threadIdx.x;
        A_ = decay;
        ag = (quad<A>*)lds;
        da = ag + quads * 64u;
        st = (A*)(da + quads * 64u);
        bc = st + 2 * SCAN_CHUNK * 64;
        l = lane_channel<LG>(p, blockIdx.y, lane);
        states_from(p, l, lane, da, (const A*)nullptr);
        sk = skip ? skip[l.ch] : A(0);
        bi = bias ? bias[l.ch] : A(0);
        dskip = dbias = A(0);
    }
    // rows [from, from + n) of a region that starts at `start`, from a multiple of 8 rows behind it; ag holds what the rows behind send
    __device__ __forceinline__ void rows(const scan_shape& p, const scan_bshape& bp, unsigned start, unsigned from, unsigned n, const scan_rows_in<T>& in,
                                         const scan_rows_out<T>& to, const scan_out<A>& out)
    {
        if (!n) return;
        scan_raw<T, LG, GATED> raw;
        unsigned c = (n - 1u) / SCAN_CHUNK;
        raw.fetch(p, bp, l, lane, n - c * SCAN_CHUNK, from + c * SCAN_CHUNK, in);
        for (;;) {
            const unsigned at = from + c * SCAN_CHUNK, chunk = (at - start) / SCAN_CHUNK;
            scan_chunk_bprop<T, LG, GATED>(p, bp, l, lane, min(SCAN_CHUNK, n - c * SCAN_CHUNK), at, in, A_, sk, bi, chunk ? kept_at(p, in.keep, start, chunk) : (const A*)nullptr,
                                    ag, da, st, bc, raw, c ? SCAN_CHUNK : 0u, to, out, dskip, dbias);
            if (c-- == 0) break;
        }
    }
    __device__ __forceinline__ void leave(const scan_shape& p, A* part)
    {
        states_to(p, l, lane, da, part);
        if (!l.active) return;
        part[(size_t)p.S * p.D + l.ch] = dskip;
        part[(size_t)(p.S + 1u) * p.D + l.ch] = dbias;
    }
};
// (shares of a group's tiles lie one behind another)
template <int LG, typename A> __device__ __forceinline__ scan_out<A> tile_share(const scan_shape& p, scan_out<A> out, size_t tile_stride)
{
    if (LG == 64) {
        const size_t o = (size_t)(blockIdx.y % p.tpg) * tile_stride;
        out.dB += o;
        out.dC += o;
    }
    return out;
}

// A wave per tile of channels takes its share of the regions one after another, with dA in LDS, and leaves one block of sums:
// part[unit][S + 2][D]. Of a region that is cut it takes the last segment, behind which nothing sends anything. Units from unit0 on
// take the other segments: the slot of segment k stands for segment k - 1, to which segment k sends what lies in the slot's carry.
template <typename T, int LG, bool GATED>
__global__ __launch_bounds__(64, sizeof(T) == 8 ? 1 : 2) void k_scan_bprop(scan_shape p, scan_bshape bp, unsigned unit0, unsigned nslot, scan_rows_in<T> in,
                                                      const typename acc_of<T>::type* __restrict__ A_, const typename acc_of<T>::type* __restrict__ skip,
                                                      const typename acc_of<T>::type* __restrict__ bias, scan_rows_out<T> to,
                                                      scan_out<typename acc_of<T>::type> out, size_t tile_stride, typename acc_of<T>::type* __restrict__ part,
                                                      const typename acc_of<T>::type* __restrict__ carry)
{
    typedef typename acc_of<T>::type A;
    extern __shared__ char lds_raw[];
    scan_wave<T, LG, GATED> w(p, lds_raw, A_, skip, bias);
    out = tile_share<LG>(p, out, tile_stride);
    const bool slots = blockIdx.x >= unit0;
    const unsigned step = slots ? gridDim.x - unit0 : unit0, stop = slots ? nslot : p.nregion;
    for (unsigned i = slots ? blockIdx.x - unit0 : blockIdx.x; i < stop; i += step) {
        row_range g;
        unsigned from, n;
        const A* sent = nullptr;
        if (slots) {
            unsigned r, k;
            if (!cut_segment(p, in.regions, in.marks, i, r, g, k)) continue;
            from = g.start + (k - 1u) * p.seg;
            n = p.seg;
            sent = carry + (size_t)i * p.S * p.D;
        } else {
            g = region_rows(in.regions, i, p.N);
            if (g.start == g.end) continue;
            from = g.start + (in.marks && is_cut(p, g) ? (g.end - g.start - 1u) / p.seg * p.seg : 0u);
            n = g.end - from;
        }
        // (a lane without a channel adds nothing to its group's sums: it has no steps, rows or states, and nothing is sent to it)
        states_from(p, w.l, w.lane, w.ag, w.l.active ? sent : (const A*)nullptr);
        w.rows(p, bp, g.start, from, n, in, to, out);
    }
    w.leave(p, part + (size_t)blockIdx.x * (p.S + 2u) * p.D);
}

// What a segment behind the first sends back when nothing is sent to it, and the sum of its steps: the states' gradients alone.
template <typename T, int LG, int NS>
__global__ __launch_bounds__(64) void k_scan_bprop_local(scan_shape p, size_t lddy, scan_rows_in<T> in, const typename acc_of<T>::type* __restrict__ A_,
                                                         const typename acc_of<T>::type* __restrict__ bias, typename acc_of<T>::type* __restrict__ local,
                                                         typename acc_of<T>::type* __restrict__ sums)
{
    typedef typename acc_of<T>::type A;
    typedef scan_weights<A, LG, NS, false, true> weights;
    constexpr unsigned U = SCAN_AHEAD;
    __shared__ A lds[weights::SIZE];
    unsigned r, k;
    row_range g;
    if (!cut_segment(p, in.regions, in.marks, blockIdx.x, r, g, k)) return;
    const scan_lane l = lane_channel<LG>(p, blockIdx.y, threadIdx.x);
    const A bi = bias ? bias[l.ch] : A(0);
    A a2[NS], ag[NS], steps = 0;
    regs_from(p, l, a2, A_, A(1.4426950408889634));
    regs_from(p, l, ag, (const A*)nullptr, A(1));
    const size_t row = (size_t)g.start + (size_t)k * p.seg;
    const unsigned place = opaque(l.ch * (unsigned)sizeof(T));
    const unsigned n = min(p.seg, g.end - (unsigned)row), up = (n + U - 1u) / U * U;
    weights w(p, threadIdx.x, first_group<LG>(p, blockIdx.y), (const A*)nullptr, in.C + row * p.ldc, lds, up - U, true);
    T dn[U], en[U], gn[U];
    auto fetch = [&](unsigned t) {               // rows t .. t + U - 1 of the segment (behind its last row: that one again)
#pragma unroll
        for (unsigned i = 0; i < U; ++i) {
            const size_t at = row + min(t + i, n - 1u);
            dn[i] = lane_load(in.dt + at * p.lddt, place);
            en[i] = lane_load(in.dY + at * lddy, place);
            if (in.gate) gn[i] = lane_load(in.gate + at * p.ldg, place);
        }
        w.fetch(n - t);
    };
    fetch(up - U);
    for (unsigned left = up; left > 0; left -= U) {
        A d[U], e[U];
#pragma unroll
        for (unsigned i = 0; i < U; ++i) {
            A slope;
            d[i] = step_of(p, (A)dn[i] + bi, slope);
            e[i] = (A)en[i];
            if (left - U + i >= n) d[i] = e[i] = A(0);
            if (in.gate) { const A gg = (A)gn[i]; e[i] *= gg * sigmoid_of(gg); }
        }
        w.put();
        if (left > U) fetch(left - 2u * U);
#pragma unroll
        for (int i = U - 1; i >= 0; --i) {
#pragma unroll
            for (int q = 0; q < NS; q += 4) {
                const quad<A> c = w.c(i, q);
#pragma unroll
                for (int j = 0; j < 4; ++j) ag[q + j] = exp2_fast(d[i] * a2[q + j]) * fma_a(c.v[j], e[i], ag[q + j]);
            }
            steps += d[i];
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    regs_to(p, l, ag, local + (size_t)blockIdx.x * p.S * p.D);
    if (l.active) sums[(size_t)blockIdx.x * p.D + l.ch] = steps;
}

// carry[slot of segment k]: what segment k >= 1 of a cut region sends to the one before it, from the last segment to the first: what it sends
// by itself, and exp(A * sum of its steps) times what it is sent. Loads run ahead of the chain.
template <typename A>
__global__ __launch_bounds__(256) void k_scan_carry_back(scan_shape p, const uint32_t* __restrict__ regions, const A* __restrict__ A_,
                                                         const A* __restrict__ local, const A* __restrict__ sums, A* __restrict__ carry)
{
    const row_range g = region_rows(regions, blockIdx.x, p.N);
    if (!is_cut(p, g)) return;
    const size_t block = (size_t)p.S * p.D, zero = g.start / p.seg;
    const unsigned n = (g.end - g.start - 1u) / p.seg;             // the last segment
    for (size_t at = (size_t)blockIdx.y * 256u + threadIdx.x; at < block; at += (size_t)gridDim.y * 256u)
        carry_chain<A>(A_[at] * A(1.4426950408889634), A(0), n, local + (zero + n) * block + at, sums + (zero + n) * p.D + at % p.D, carry + (zero + n) * block + at,
                       0 - block, 0 - (size_t)p.D);
}

// dB and dC from the tiles' shares, in the tiles' order: a region's rows (its first segment's where it is cut), or another segment's.
template <typename A>
__global__ __launch_bounds__(256) void k_scan_weights(scan_shape p, const uint32_t* __restrict__ regions, const uint32_t* __restrict__ marks, unsigned tiles,
                                                      size_t ncol, const A* __restrict__ share, size_t tile_stride, A* __restrict__ dB, size_t lddb, A* __restrict__ dC, size_t lddc)
{
    row_range g;
    unsigned from;
    if (blockIdx.x < p.nregion) {
        g = region_rows(regions, blockIdx.x, p.N);
        from = g.start;
        if (marks && is_cut(p, g)) g.end = g.start + p.seg;
    } else {
        unsigned r, k;
        if (!cut_segment(p, regions, marks, blockIdx.x - p.nregion, r, g, k)) return;
        from = g.start + k * p.seg;
        g.end = min(g.end, from + p.seg);
    }
    const size_t n = (size_t)(g.end - from) * 2u * ncol;
    for (size_t i = (size_t)blockIdx.y * 256u + threadIdx.x; i < n; i += (size_t)gridDim.y * 256u) {
        const size_t row = from + i / (2u * ncol), c = i % (2u * ncol);
        A s = 0;
#pragma unroll 4
        for (unsigned t = 0; t < tiles; ++t) s += share[t * tile_stride + row * 2u * ncol + c];
        if (c < ncol) dB[row * lddb + c] = s;
        else dC[row * lddc + c - ncol] = s;
    }
}

namespace {

constexpr size_t SCAN_UNITS = 4096;              // waves that add up dA, over all tiles of channels: four per SIMD that the chip has room for
constexpr size_t SCAN_WAVES = 2048;              // waves that keep the vector units busy: two per SIMD, which 256 registers a lane allow
constexpr size_t SCAN_LEAST = 32;                // rows of the shortest segment

scan_plan plan_bprop(const dbk_statescan_args& a) { return plan_scan(a.N, a.D, a.G, SCAN_WAVES, 2, SCAN_LEAST); }

// Workspace: segments, tiles' shares of dB and dC (a group of several tiles), units' sums of dA, dD and dbias.
struct bprop_layout { scan_segments seg; size_t share, part, bytes; unsigned units, slot_units; };
bprop_layout layout_of(void* work, const dbk_statescan_args& a, const scan_plan& p)
{
    bprop_layout y;
    const size_t e = acc_size(a.dtype), cap = SCAN_UNITS / p.tiles ? SCAN_UNITS / p.tiles : 1;
    y.units = (unsigned)(a.nregion < cap ? a.nregion : cap);
    y.slot_units = (unsigned)(p.slots < cap ? p.slots : cap);
    y.seg = segments_in(work, a, p);
    y.share = y.seg.bytes;
    y.part = y.share + (p.tpg > 1 ? ((size_t)p.tpg * a.N * 2 * a.G * a.S * e + 15) / 16 * 16 : 0);
    y.bytes = y.part + (size_t)(y.units + y.slot_units) * (a.S + 2) * a.D * e;
    return y;
}

// Workgroups per region or segment that add the tiles' shares, four values a thread: as many as a whole segment has work for where there are few of them, what the
// average has where there are many, whose sum would otherwise be workgroups without work (20 thousand reads x 256 channels: 97 of 100, 11.9 ms a pass instead of 11.3).
unsigned weights_blocks(const dbk_statescan_args& a, const scan_plan& p)
{
    const size_t per_row = 2 * a.G * a.S, items = a.nregion + p.slots, most = ((size_t)p.seg * per_row + 1023) / 1024;
    const size_t average = a.N * per_row / items / 1024 + 1, room = 65536 / items + 1, want = average > room ? average : room;
    const size_t wgs = want < most ? want : most;
    return (unsigned)(wgs < 65535 ? wgs : 65535);
}

}  // namespace

size_t bprop_work_bytes(const dbk_statescan_args& a) { return layout_of(nullptr, a, plan_bprop(a)).bytes; }

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
    const scan_plan p = plan_bprop(*a);
    const bprop_layout y = layout_of(work, *a, p);
    DBK_CHECK(grid_fits(a->nregion + p.slots, 256), "ValueError: map too large (%zu rows, %zu regions)", a->N, a->nregion);
    DBK_CHECK(work && work_bytes >= y.bytes, "ValueError: the workspace has %zu bytes, %zu are needed", work_bytes, y.bytes);
    const scan_shape s = shape_of(*a, p);
    const scan_bshape b = {a->lddy, a->lddx, a->ldddt, a->lddgate, a->lddb, a->lddc};
    const size_t ncol = a->G * a->S;
    const bool shared = p.tpg > 1;
    void* part = (char*)work + y.part;
    if (p.slots) mark_cut_regions(st, s, a->regions, y.seg.marks);
    with_row_type(a->dtype, [&](auto t) {
        typedef decltype(t) T;
        typedef typename acc_of<T>::type A;
        A* share = (A*)((char*)work + y.share);
        const size_t tile_stride = shared ? a->N * 2 * ncol : 0;                // a tile's share: (N, dB | dC)
        const scan_out<A> out = shared ? scan_out<A>{share, share + ncol, 2 * ncol, 2 * ncol} : scan_out<A>{(A*)a->dB, (A*)a->dC, a->lddb, a->lddc};
        const scan_rows_in<T> in = {(const T*)a->X, (const T*)a->dt, (const T*)a->gate, (const T*)a->dY, (const A*)a->B, (const A*)a->C, (const A*)a->keep, a->regions, y.seg.marks};
        const scan_rows_out<T> to = {(T*)a->dX, (T*)a->ddt, (T*)a->dgate};
        const size_t quads = (a->S + 3) / 4, pad = a->S <= 16 ? 16 : quads * 4;
        const size_t lds = quads * 64 * 2 * sizeof(quad<A>) + (2 * 64 + 2 * (64 / p.lanes) * pad) * SCAN_CHUNK * sizeof(A);
        with_lanes(p.lanes, [&](auto lanes) {
            if (p.slots) {
                with_states(a->S, [&](auto ns) {
                    k_scan_bprop_local<T, lanes.value, ns.value><<<dim3(p.slots, p.tiles), 64, 0, st>>>(s, b.lddy, in, (const A*)a->A, (const A*)a->dt_bias,
                                                                                                        (A*)y.seg.local, (A*)y.seg.steps);
                });
                k_scan_carry_back<A><<<dim3((unsigned)a->nregion, carry_blocks(*a)), 256, 0, st>>>(s, a->regions, (const A*)a->A, (const A*)y.seg.local,
                                                                                                  (const A*)y.seg.steps, (A*)y.seg.carry);
            }
            auto main = [&](auto gated) {
                k_scan_bprop<T, lanes.value, gated.value><<<dim3(y.units + y.slot_units, p.tiles), 64, lds, st>>>(
                    s, b, y.units, p.slots, in, (const A*)a->A, (const A*)a->skip, (const A*)a->dt_bias, to, out, tile_stride, (A*)part, (const A*)y.seg.carry);
            };
            if (a->gate) main(std::true_type());
            else main(std::false_type());
        });
        if (shared)
            k_scan_weights<A><<<dim3((unsigned)a->nregion + p.slots, weights_blocks(*a, p)), 256, 0, st>>>(s, a->regions, y.seg.marks, p.tpg, ncol, share, tile_stride,
                                                                                                      (A*)a->dB, a->lddb, (A*)a->dC, a->lddc);
    });
    sum_partials(st, a->dtype, part, y.units + y.slot_units, a->S * a->D, a->dA, a->D, a->dskip, a->D, a->ddt_bias);
    DBK_LAUNCH_OK();
}

}  // extern "C"
