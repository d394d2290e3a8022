// The norms around a block of layers, with the block's gate and residual, forward and backward: y is what the block makes, r the residual that goes past it.
//
//   p = norm(y) gamma + beta,  r' = r + scale p g sigmoid(g),  z = norm(r') next_gamma + next_beta
//
// norm(x) = (x - mean) / sqrt(mean((x - mean)^2) + eps) over a chunk of a row, or x / sqrt(mean(x^2) + eps) (rms). Every part may be left out. The second
// norm is of r' as it is kept, which is what the next block and the backward pass see. With h1 = norm(y), h2 = norm(r') and the gradients dr (of r' from elsewhere) and dz:
//
//   t = dr + back(dz next_gamma, h2),  back(q, h) = rstd (q - mean(q) - h mean(q h))  (rms: without mean(q))
//   dr_in = t,  dp = t scale g sigmoid(g),  dy = back(dp gamma, h1),  dg = t scale p (sigmoid(g) (1 + g (1 - sigmoid(g))))
//   dgamma = sum dp h1,  dbeta = sum dp,  dscale = sum t p g sigmoid(g),  dnext_gamma = sum dz h2,  dnext_beta = sum dz
//
// Bound by memory: forward three maps in and two out, backward five in and three out. A thread holds one vector of 16 bytes of a chunk, a chunk belongs to a power of two
// of a wave's lanes, or to a workgroup of two to sixteen waves, and a workgroup walks down the rows with its chunks' weights, and backward their gradients, in registers.
// 50 021 rows x 64 chunks of 16 floats, rms, no gate: 160 us forward (820 MB, 5.1 TB/s), 252 backward (1230 MB, 4.9) and 8 for the sums; 130 003 rows x 1440 bfloat16 with a gate: 417
// (1870 MB, 4.5 TB/s; vector instructions 74 % of the time: two norms, a sigmoid and conversions for ten bytes) and 622 (2996 MB, 4.8; three barriers a row), once the clocks have settled: the
// first dozen passes after a pause take 440 to 500 and 650 to 760.
#include <type_traits>
#include "norm_common.h"

namespace dbk {

struct block_shape {
    unsigned n, nchunk, width, ct_log2, rstep;
    int rms, norm, next;                         // rms norms; whether y, and r', are normalised
    size_t ldy, ldr, ldg, ldo, ldz;              // y, r, gate; r' and z
    size_t lddr, lddz, lddy, lddo, lddg;         // backward: dr and dz in, dy, dr and dgate out (ldo: r')
};

// sums over LANES lanes of two values at once
template <int LANES, typename A> __device__ __forceinline__ void block_sum2(A& u, A& v, A (*lds)[16])
{
    if constexpr (LANES >= 16) {
        u += rotated<8>(u); v += rotated<8>(v);
        u += rotated<4>(u); v += rotated<4>(v);
        u += rotated<2>(u); v += rotated<2>(v);
        u += rotated<1>(u); v += rotated<1>(v);
        constexpr int W = LANES < 64 ? LANES : 64;
#pragma unroll
        for (int o = 16; o < W; o *= 2) {
            u += __shfl_xor(u, o);
            v += __shfl_xor(v, o);
        }
    } else
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) {
            u += __shfl_xor(u, o);
            v += __shfl_xor(v, o);
        }
    if constexpr (LANES > 64) {
        constexpr int N = LANES / 64;
        __syncthreads();                         // (the words may still be read from the sums before)
        if ((threadIdx.x & 63) == 0) { lds[0][threadIdx.x >> 6] = u; lds[1][threadIdx.x >> 6] = v; }
        __syncthreads();
        u = v = A(0);
#pragma unroll
        for (int w = 0; w < N; ++w) { u += lds[0][w]; v += lds[1][w]; }
    }
}

// mean and reciprocal deviation of a chunk whose values lie in x
template <int LANES, typename A, int V> __device__ __forceinline__ void chunk_stats(const A (&x)[V], unsigned valid, A inv, A eps, bool rms, A& mean, A& rstd, A (*lds)[16])
{
    A a = A(0), b = A(0);
    if (rms) {
#pragma unroll
        for (int j = 0; j < V; ++j) a = fma(x[j], x[j], a);      // (zeros behind the last)
        block_sum2<LANES>(a, b, lds);
        mean = A(0);
        rstd = A(1) / sqrt(a * inv + eps);
        return;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) a += x[j];
    block_sum2<LANES>(a, b, lds);
    const A near = a * inv;
    a = b = A(0);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const A c = j < (int)valid ? x[j] - near : A(0);
        a = fma(c, c, a);
        b += c;
    }
    block_sum2<LANES>(a, b, lds);
    norm_stats(near, a * inv, b * inv, eps, mean, rstd);
}

template <int LANES> constexpr int block_threads() { return LANES > 64 ? LANES : 256; }

// Where a thread's vector lies: LANES lanes of a chunk; up to 64 lanes several chunks or rows share a workgroup.
template <int LANES, int V> struct block_place {
    unsigned chunk, lane, valid, first, row;     // first: of the workgroup's rows
    size_t column;
    __device__ __forceinline__ block_place(const block_shape& p)
    {
        const unsigned unit = threadIdx.x / LANES;
        lane = threadIdx.x % LANES;
        chunk = (blockIdx.y << p.ct_log2) + (unit & ((1u << p.ct_log2) - 1u));
        valid = chunk < p.nchunk && lane * V < p.width ? p.width - lane * V : 0u;
        first = blockIdx.x * (block_threads<LANES>() / LANES) >> p.ct_log2;
        row = first + (unit >> p.ct_log2);
        column = (size_t)chunk * p.width + lane * V;
    }
    __device__ __forceinline__ bool leads(const block_shape& p) const { return lane == 0u && chunk < p.nchunk; }
};

// step(ahead, row) for every row of a lane, each fetched one or two (as many as `ahead` holds) of the lane's rows before. Every lane of a workgroup makes the same number of
// steps, whether its row exists or not: sums over its waves meet at barriers.
template <typename AHEAD, int N, typename FETCH, typename STEP>
__device__ __forceinline__ void walk_rows(const block_shape& p, unsigned first, size_t row, AHEAD (&ahead)[N], FETCH fetch, STEP step)
{
    const size_t by = (size_t)N * p.rstep;
#pragma unroll
    for (int i = 0; i < N; ++i) fetch(ahead[i], row + (size_t)i * p.rstep);
    for (size_t left = first; left < p.n; left += by, row += by) {
        step(ahead[0], row);
        if (N > 1 && left + p.rstep < p.n) step(ahead[N - 1], row + p.rstep);
    }
}

// LANES of more than 64 share a workgroup of their own size with no other chunk: plan_block gives it one row at a time.
template <typename T, int LANES, bool EXACT>
__global__ __launch_bounds__(block_threads<LANES>()) void k_block_fprop(block_shape p, const T* __restrict__ Y, const T* __restrict__ R, const T* __restrict__ gate,
                                                                       const typename acc_of<T>::type* __restrict__ gamma, const typename acc_of<T>::type* __restrict__ beta,
                                                                       const typename acc_of<T>::type* __restrict__ scale, const typename acc_of<T>::type* __restrict__ ngamma,
                                                                       const typename acc_of<T>::type* __restrict__ nbeta, typename acc_of<T>::type eps, T* __restrict__ O,
                                                                       T* __restrict__ Z, typename acc_of<T>::type* __restrict__ stats)
{
    typedef typename acc_of<T>::type A;
    constexpr int V = row_vec<T>::N;
    __shared__ A lds[2][16];
    const block_place<LANES, V> at(p);
    A g1[V], b1[V], sc[V], g2[V], b2[V];
    load_weights(g1, gamma ? gamma + at.column : nullptr, at.valid, A(1));
    load_weights(b1, beta ? beta + at.column : nullptr, at.valid, A(0));
    load_weights(sc, scale ? scale + at.column : nullptr, at.valid, A(1));
    load_weights(g2, ngamma ? ngamma + at.column : nullptr, at.valid, A(1));
    load_weights(b2, nbeta ? nbeta + at.column : nullptr, at.valid, A(0));
    const A inv = A(1) / (A)p.width;
    const size_t units = (size_t)p.n * p.nchunk;
    // (a second row ahead is worth 170 to 158 us on 50021 rows of 64 chunks of 16 floats; bfloat16 ones it costs a fourth wave per SIMD: 491 us for 435 on 130003 x 1440)
    constexpr unsigned AHEAD = sizeof(T) == 2 ? 1 : 2;
    struct { raw_vec<T, EXACT> y, r, g; } ahead[AHEAD];
    auto fetch = [&](auto& to, size_t row) {
        const unsigned valid = row < p.n ? at.valid : 0u;
        to.y.load(Y + row * p.ldy + at.column, valid);
        if (R) to.r.load(R + row * p.ldr + at.column, valid);
        if (gate) to.g.load(gate + row * p.ldg + at.column, valid);
    };
    auto step = [&](auto& from, size_t now) {
        const raw_vec<T, EXACT> y = from.y, r = from.r, g = from.g;
        fetch(from, now + AHEAD * (size_t)p.rstep);
        A x[V], mean = A(0), rstd = A(1);
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = y[j];
        if (p.norm) chunk_stats<LANES>(x, at.valid, inv, eps, p.rms, mean, rstd, lds);
        if (stats && now < p.n && at.leads(p)) {
            stats[(size_t)now * p.nchunk + at.chunk] = mean;
            stats[units + (size_t)now * p.nchunk + at.chunk] = rstd;
        }
        row_vec<T> o;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            A v = fma((x[j] - mean) * rstd, g1[j], b1[j]) * sc[j];
            if (gate) v *= g[j] * sigmoid_of(g[j]);
            if (R) v += r[j];
            x[j] = j < (int)at.valid ? (A)(T)v : A(0);           // (as it is kept)
            o.v[j] = v;
        }
        const bool here = now < p.n;
        store_vec<EXACT>(o, O + now * p.ldo + at.column, here ? at.valid : 0u);
        if (!p.next) return;
        chunk_stats<LANES>(x, at.valid, inv, eps, p.rms, mean, rstd, lds);
        if (stats && here && at.leads(p)) {
            stats[2 * units + (size_t)now * p.nchunk + at.chunk] = mean;
            stats[3 * units + (size_t)now * p.nchunk + at.chunk] = rstd;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) o.v[j] = fma((x[j] - mean) * rstd, g2[j], b2[j]);
        store_vec<EXACT>(o, Z + now * p.ldz + at.column, here ? at.valid : 0u);
    };
    walk_rows(p, at.first, at.row, ahead, fetch, step);
}

// The weights' gradients of a workgroup's rows are added in registers, its row lanes in LDS at the end, in a fixed order: part[blockIdx.x][5][m].
template <typename T, int LANES, bool EXACT, bool RMS>
__global__ __launch_bounds__(block_threads<LANES>()) void k_block_bprop(block_shape p, const T* __restrict__ Y, const T* __restrict__ O, const T* __restrict__ gate,
                                                                       const typename acc_of<T>::type* __restrict__ gamma, const typename acc_of<T>::type* __restrict__ beta,
                                                                       const typename acc_of<T>::type* __restrict__ scale, const typename acc_of<T>::type* __restrict__ ngamma,
                                                                       const typename acc_of<T>::type* __restrict__ stats, const T* __restrict__ dR, const T* __restrict__ dZ,
                                                                       T* __restrict__ dY, T* __restrict__ dO, T* __restrict__ dgate, typename acc_of<T>::type* __restrict__ part)
{
    typedef typename acc_of<T>::type A;
    constexpr int V = row_vec<T>::N;
    __shared__ A lds[2][16];
    __shared__ A strips[LANES <= 64 ? 256 : 1][V + 1];
    const block_place<LANES, V> at(p);
    A g1[V], b1[V], sc[V], g2[V], sums[5][V];
    load_weights(g1, gamma ? gamma + at.column : nullptr, at.valid, A(1));
    load_weights(b1, beta ? beta + at.column : nullptr, at.valid, A(0));
    load_weights(sc, scale ? scale + at.column : nullptr, at.valid, A(1));
    load_weights(g2, ngamma ? ngamma + at.column : nullptr, at.valid, A(1));
#pragma unroll
    for (int i = 0; i < 5; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) sums[i][j] = A(0);
    const A inv = A(1) / (A)p.width;
    const size_t units = (size_t)p.n * p.nchunk;
    // (a second row ahead costs float rows two of four waves per SIMD: 262 us where it is 247 on 50021 rows of 64 chunks; bfloat16 ones nothing: 744 for 857 on 130003 x 1440)
    constexpr unsigned AHEAD = sizeof(T) == 2 ? 2 : 1;
    struct { raw_vec<T, EXACT> y, o, g, d, z; A s[4]; } ahead[AHEAD];
    auto fetch = [&](auto& to, size_t row) {
        const bool here = row < p.n && at.chunk < p.nchunk;
        const unsigned valid = here ? at.valid : 0u;
        const size_t u = row * p.nchunk + at.chunk;
        to.y.load(Y + row * p.ldy + at.column, valid);
        if (gate) to.g.load(gate + row * p.ldg + at.column, valid);
        to.d.load(dR + row * p.lddr + at.column, dR ? valid : 0u);
        if (p.norm) { to.s[0] = here && !RMS ? stats[u] : A(0); to.s[1] = here ? stats[units + u] : A(0); }
        if (p.next) {
            to.o.load(O + row * p.ldo + at.column, valid);
            to.z.load(dZ + row * p.lddz + at.column, valid);
            to.s[2] = here && !RMS ? stats[2 * units + u] : A(0);
            to.s[3] = here ? stats[3 * units + u] : A(0);
        }
    };
    auto step = [&](auto& from, size_t now) {
        const raw_vec<T, EXACT> y = from.y, o = from.o, g = from.g, d = from.d, z = from.z;
        const A mean1 = p.norm ? from.s[0] : A(0), rstd1 = p.norm ? from.s[1] : A(1), mean2 = from.s[2], rstd2 = from.s[3];
        fetch(from, now + AHEAD * (size_t)p.rstep);
        const bool here = now < p.n;
        // (lanes and rows that do not exist send nothing back: t is zero there, and with it all that follows)
        A t[V], a = A(0), b = A(0);
        if (p.next) {
            A h[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                h[j] = RMS ? o[j] * rstd2 : (o[j] - mean2) * rstd2;
                t[j] = z[j] * g2[j];
                sums[3][j] = fma(z[j], h[j], sums[3][j]);
                sums[4][j] += z[j];
                if (!RMS) a += t[j];
                b = fma(t[j], h[j], b);
            }
            block_sum2<LANES>(a, b, lds);
            a = RMS ? A(0) : a * inv;
            b *= -inv;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const A q = fma(h[j], b, RMS ? t[j] : t[j] - a);
                t[j] = (EXACT ? at.valid != 0u : j < (int)at.valid) && here ? fma(rstd2, q, d[j]) : A(0);
            }
        } else
#pragma unroll
            for (int j = 0; j < V; ++j) t[j] = d[j];
        row_vec<T> out;
        if (dO) {
#pragma unroll
            for (int j = 0; j < V; ++j) out.v[j] = t[j];
            store_vec<EXACT>(out, dO + now * p.lddo + at.column, here ? at.valid : 0u);
        }
        A q[V];
        a = b = A(0);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const A h = RMS ? y[j] * rstd1 : (y[j] - mean1) * rstd1, pv = RMS && !beta ? h * g1[j] : fma(h, g1[j], b1[j]), ts = t[j] * sc[j], tp = t[j] * pv;
            A dp = ts;
            if (gate) {
                const A e = sigmoid_of(g[j]), act = g[j] * e;
                dp = ts * act;
                out.v[j] = ts * pv * fma(act, A(1) - e, e);
                sums[2][j] = fma(tp, act, sums[2][j]);
            } else
                sums[2][j] += tp;
            sums[0][j] = fma(dp, h, sums[0][j]);
            sums[1][j] += dp;
            q[j] = dp * g1[j];
            if (!RMS) a += q[j];
            b = fma(q[j], h, b);
        }
        if (gate) store_vec<EXACT>(out, dgate + now * p.lddg + at.column, here ? at.valid : 0u);
        if (p.norm) {
            block_sum2<LANES>(a, b, lds);
            a = RMS ? A(0) : a * inv;
            b *= -inv;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const A h = RMS ? y[j] * rstd1 : (y[j] - mean1) * rstd1;
                out.v[j] = rstd1 * fma(h, b, RMS ? q[j] : q[j] - a);
            }
        } else
#pragma unroll
            for (int j = 0; j < V; ++j) out.v[j] = q[j];
        store_vec<EXACT>(out, dY + now * p.lddy + at.column, here ? at.valid : 0u);
    };
    walk_rows(p, at.first, at.row, ahead, fetch, step);
    if (!part) return;
    const size_t m = (size_t)p.nchunk * p.width;
    const unsigned across = LANES << p.ct_log2;                 // threads of one row lane
#pragma unroll
    for (int i = 0; i < 5; ++i) {
        if constexpr (LANES <= 64) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < V; ++j) strips[threadIdx.x][j] = sums[i][j];
            sum_strips(strips, across, V);
        }
        if (threadIdx.x >= across || !at.valid) continue;
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (j < (int)at.valid) part[((size_t)blockIdx.x * 5u + i) * m + at.column + j] = LANES <= 64 ? strips[LANES <= 64 ? threadIdx.x : 0][j] : sums[i][j];
    }
}

// Chunks too wide for a workgroup's threads: a workgroup per chunk goes over it once per sum (from the caches after the first time).
constexpr int WIDE = 1024;

template <typename T, typename F> __device__ __forceinline__ void wide_stats(unsigned width, typename acc_of<T>::type eps, bool rms, typename acc_of<T>::type& mean,
                                                                            typename acc_of<T>::type& rstd, typename acc_of<T>::type (*lds)[16], F value)
{
    typedef typename acc_of<T>::type A;
    const A inv = A(1) / (A)width;
    A a = A(0), b = A(0);
    for (unsigned c = threadIdx.x; c < width; c += WIDE) { const A x = value(c); a += rms ? x * x : x; }
    block_sum2<WIDE>(a, b, lds);
    if (rms) { mean = A(0); rstd = A(1) / sqrt(a * inv + eps); return; }
    const A near = a * inv;
    a = b = A(0);
    for (unsigned c = threadIdx.x; c < width; c += WIDE) { const A x = value(c) - near; a = fma(x, x, a); b += x; }
    block_sum2<WIDE>(a, b, lds);
    norm_stats(near, a * inv, b * inv, eps, mean, rstd);
}

template <typename T>
__global__ __launch_bounds__(WIDE) void k_block_fprop_wide(block_shape p, const T* __restrict__ Y, const T* __restrict__ R, const T* __restrict__ gate,
                                                           const typename acc_of<T>::type* __restrict__ gamma, const typename acc_of<T>::type* __restrict__ beta,
                                                           const typename acc_of<T>::type* __restrict__ scale, const typename acc_of<T>::type* __restrict__ ngamma,
                                                           const typename acc_of<T>::type* __restrict__ nbeta, typename acc_of<T>::type eps, T* O, T* __restrict__ Z,
                                                           typename acc_of<T>::type* __restrict__ stats)
{
    typedef typename acc_of<T>::type A;
    __shared__ A lds[2][16];
    const size_t units = (size_t)p.n * p.nchunk;
    for (size_t u = blockIdx.x; u < units; u += gridDim.x) {
        const size_t row = u / p.nchunk, col = u % p.nchunk * p.width;
        const T *y = Y + row * p.ldy + col, *r = R ? R + row * p.ldr + col : nullptr, *g = gate ? gate + row * p.ldg + col : nullptr;
        T *o = O + row * p.ldo + col, *z = Z ? Z + row * p.ldz + col : nullptr;
        A mean = A(0), rstd = A(1);
        if (p.norm) wide_stats<T>(p.width, eps, p.rms, mean, rstd, lds, [&](unsigned c) { return (A)y[c]; });
        for (unsigned c = threadIdx.x; c < p.width; c += WIDE) {
            A v = fma(((A)y[c] - mean) * rstd, gamma ? gamma[col + c] : A(1), beta ? beta[col + c] : A(0)) * (scale ? scale[col + c] : A(1));
            if (g) v *= (A)g[c] * sigmoid_of((A)g[c]);
            if (r) v += (A)r[c];
            o[c] = (T)v;
        }
        if (stats && threadIdx.x == 0) { stats[u] = mean; stats[units + u] = rstd; }
        if (!p.next) continue;
        // (a thread reads the values of r' that it wrote itself)
        wide_stats<T>(p.width, eps, p.rms, mean, rstd, lds, [&](unsigned c) { return (A)o[c]; });
        for (unsigned c = threadIdx.x; c < p.width; c += WIDE)
            z[c] = (T)fma(((A)o[c] - mean) * rstd, ngamma ? ngamma[col + c] : A(1), nbeta ? nbeta[col + c] : A(0));
        if (stats && threadIdx.x == 0) { stats[2 * units + u] = mean; stats[3 * units + u] = rstd; }
    }
}

// What one value of r' and y sends back, given its chunk's sums: t and what the weights' gradients take
template <typename A> struct block_value {
    A t, h1, h2, p, act, open;                   // open: the gate's derivative
    __device__ __forceinline__ void of(const block_shape& s, A y, A o, A g, bool gated, A d, A z, A g1, A b1, A g2, A mean1, A rstd1, A mean2, A rstd2, A a, A b)
    {
        h1 = (y - mean1) * rstd1;
        h2 = s.next ? (o - mean2) * rstd2 : A(0);
        t = d;
        if (s.next) t += rstd2 * (fma(z, g2, -a) - h2 * b);
        p = fma(h1, g1, b1);
        act = open = A(1);
        if (gated) { const A e = sigmoid_of(g); act = g * e; open = e * fma(g, A(1) - e, A(1)); }
    }
};

template <typename T>
__global__ __launch_bounds__(WIDE) void k_block_bprop_wide(block_shape p, const T* __restrict__ Y, const T* __restrict__ O, const T* __restrict__ gate,
                                                           const typename acc_of<T>::type* __restrict__ gamma, const typename acc_of<T>::type* __restrict__ beta,
                                                           const typename acc_of<T>::type* __restrict__ scale, const typename acc_of<T>::type* __restrict__ ngamma,
                                                           const typename acc_of<T>::type* __restrict__ stats, const T* __restrict__ dR, const T* __restrict__ dZ, T* __restrict__ dY,
                                                           T* __restrict__ dO, T* __restrict__ dgate, typename acc_of<T>::type* __restrict__ part)
{
    typedef typename acc_of<T>::type A;
    __shared__ A lds[2][16];
    const size_t units = (size_t)p.n * p.nchunk, m = (size_t)p.nchunk * p.width;
    const A inv = A(1) / (A)p.width;
    // chunk by chunk, each workgroup rows of its own: a thread's columns are always the same, and it adds its rows to its own partial sums
    for (unsigned chunk = 0; chunk < p.nchunk; ++chunk) {
        const size_t col = (size_t)chunk * p.width;
        bool before = false;
        for (size_t row = blockIdx.x; row < p.n; row += gridDim.x) {
            const size_t u = row * p.nchunk + chunk;
            const T *y = Y + row * p.ldy + col, *o = p.next ? O + row * p.ldo + col : nullptr, *g = gate ? gate + row * p.ldg + col : nullptr;
            const T *d = dR ? dR + row * p.lddr + col : nullptr, *z = p.next ? dZ + row * p.lddz + col : nullptr;
            const A mean1 = p.norm ? stats[u] : A(0), rstd1 = p.norm ? stats[units + u] : A(1), mean2 = p.next ? stats[2 * units + u] : A(0), rstd2 = p.next ? stats[3 * units + u] : A(0);
            A a = A(0), b = A(0), a1 = A(0), b1 = A(0);
            if (p.next) {
                for (unsigned c = threadIdx.x; c < p.width; c += WIDE) {
                    const A q = (A)z[c] * (ngamma ? ngamma[col + c] : A(1));
                    a += q;
                    b = fma(q, ((A)o[c] - mean2) * rstd2, b);
                }
                block_sum2<WIDE>(a, b, lds);
                a = p.rms ? A(0) : a * inv;
                b *= inv;
            }
            auto value = [&](unsigned c) {
                block_value<A> v;
                v.of(p, (A)y[c], p.next ? (A)o[c] : A(0), g ? (A)g[c] : A(0), g != nullptr, d ? (A)d[c] : A(0), p.next ? (A)z[c] : A(0), gamma ? gamma[col + c] : A(1),
                     beta ? beta[col + c] : A(0), ngamma ? ngamma[col + c] : A(1), mean1, rstd1, mean2, rstd2, a, b);
                return v;
            };
            if (p.norm) {
                for (unsigned c = threadIdx.x; c < p.width; c += WIDE) {
                    const block_value<A> v = value(c);
                    const A q = v.t * (scale ? scale[col + c] : A(1)) * v.act * (gamma ? gamma[col + c] : A(1));
                    a1 += q;
                    b1 = fma(q, v.h1, b1);
                }
                block_sum2<WIDE>(a1, b1, lds);
                a1 = p.rms ? A(0) : a1 * inv;
                b1 *= inv;
            }
            for (unsigned c = threadIdx.x; c < p.width; c += WIDE) {
                const block_value<A> v = value(c);
                const A ts = v.t * (scale ? scale[col + c] : A(1)), dp = ts * v.act, q = dp * (gamma ? gamma[col + c] : A(1));
                dY[row * p.lddy + col + c] = (T)(p.norm ? rstd1 * (q - a1 - v.h1 * b1) : q);
                if (dO) dO[row * p.lddo + col + c] = (T)v.t;
                if (g) dgate[row * p.lddg + col + c] = (T)(ts * v.p * v.open);
                if (!part) continue;
                A* s = part + (size_t)blockIdx.x * 5u * m + col + c;
                const A zc = p.next ? (A)z[c] : A(0), more[5] = {dp * v.h1, dp, v.t * v.p * v.act, zc * v.h2, zc};
#pragma unroll
                for (int i = 0; i < 5; ++i) s[i * m] = before ? s[i * m] + more[i] : more[i];
            }
            before = true;
        }
    }
}

namespace {

struct block_plan {
    int lanes;                                   // 0: the wide kernels
    unsigned gx, gy;
    block_shape shape;
};

// Workgroups that walk the rows. Forward several rounds of waves even out (bfloat16 435 us with 8192, 483 with the 4096 that run at once); backward, where each workgroup's partial sums are
// added up afterwards, no more than run at once: three waves per SIMD with four floats a lane, two with eight bfloat16 values, three with two doubles.
inline unsigned block_wgs(int dtype, bool backward, unsigned waves)
{
    if (!backward) return 8192u / waves;
    const unsigned fit = (dtype == DBK_BF16 ? 8u : 12u) / waves;
    return 256u * (fit ? fit : 1u);
}
constexpr size_t WIDE_WGS = 512;

block_plan plan_block(const dbk_blocknorm_args& a, bool backward)
{
    block_plan p = {};
    const size_t V = 16 / row_size(a.dtype), vecs = (a.group + V - 1) / V, nchunk = a.m / a.group;
    // Six waves only backward (60 003 x 1400 floats 581 -> 555 us, x 700 doubles 828 -> 632; forward 351 -> 395, as fewer waves fit a CU), twelve both ways (40 003 x 2500 floats 434 -> 405 and
    // 639 -> 598); three gain nothing (100 003 x 700 floats 311 -> 320 and 450 -> 475). More than eight waves of bfloat16 rows backward lack registers: 50 003 x 5600 takes 3640 us with
    // twelve, 6870 with sixteen, 7220 without them at all.
    for (int lanes : {1, 2, 4, 8, 16, 32, 64, 128, 256, 384, 512, 768, 1024})
        if (!p.lanes && vecs <= (size_t)lanes && (backward || lanes != 384)) p.lanes = lanes;
    const unsigned threads = p.lanes > 64 ? p.lanes : 256u;
    const unsigned ct = p.lanes && p.lanes <= 64 ? chunks_side_by_side((unsigned)p.lanes, nchunk) : 0u;
    const unsigned rt = p.lanes ? (threads / p.lanes) >> ct : 1u;
    p.gy = p.lanes ? divup(nchunk, size_t(1) << ct) : 1u;
    const unsigned wgs = block_wgs(a.dtype, backward, threads / 64u), most = wgs / p.gy ? wgs / p.gy : 1u;
    p.gx = divup(a.n, rt);
    if (p.gx > most) p.gx = most;
    if (!p.lanes) p.gx = (unsigned)(a.n < WIDE_WGS ? a.n : WIDE_WGS);
    block_shape& s = p.shape;
    s.n = (unsigned)a.n;
    s.nchunk = (unsigned)nchunk;
    s.width = (unsigned)a.group;
    s.ct_log2 = ct;
    s.rstep = p.gx * rt;
    s.rms = a.rms;
    s.norm = a.norm;
    s.next = a.next;
    s.ldy = a.ldy; s.ldr = a.ldr; s.ldg = a.ldgate; s.ldo = a.ldo; s.ldz = a.ldz;
    s.lddr = a.lddr; s.lddz = a.lddz; s.lddy = a.lddy; s.lddo = a.lddr_in; s.lddg = a.lddgate;
    return p;
}

template <bool BACK, typename F> bool block_layout(int lanes, bool exact, F f)
{
#define DBK_BLOCK_CASE(L)                                                        \
    if constexpr (BACK || L != 384)                                                   \
        if (lanes == L) {                                                        \
            if (exact) f(std::integral_constant<int, L>(), std::true_type());    \
            else f(std::integral_constant<int, L>(), std::false_type());         \
            return true;                                                         \
        }
    DBK_BLOCK_CASE(1) DBK_BLOCK_CASE(2) DBK_BLOCK_CASE(4) DBK_BLOCK_CASE(8) DBK_BLOCK_CASE(16) DBK_BLOCK_CASE(32) DBK_BLOCK_CASE(64)
    DBK_BLOCK_CASE(128) DBK_BLOCK_CASE(256) DBK_BLOCK_CASE(384) DBK_BLOCK_CASE(512) DBK_BLOCK_CASE(768) DBK_BLOCK_CASE(1024)
#undef DBK_BLOCK_CASE
    return false;
}

int check_block(const dbk_blocknorm_args* a)
{
    DBK_CHECK(a, "ValueError: null argument block");
    DBK_ROW_DTYPE_OK(a->dtype);
    DBK_CHECK(a->group >= 1 && a->m % a->group == 0, "ValueError: the number of columns must be divisible by the chunk's");
    DBK_CHECK(a->n < (size_t(1) << 31) && a->m < (size_t(1) << 31), "ValueError: matrix too large (%zu x %zu)", a->n, a->m);
    DBK_CHECK(a->norm || (!a->gamma && !a->beta), "ValueError: weights of a norm that is left out");
    DBK_CHECK(a->next || (!a->next_gamma && !a->next_beta), "ValueError: weights of a norm that is left out");
    DBK_CHECK(!a->n || !a->m || a->Y, "ValueError: null matrix");
    DBK_CHECK(!a->m || plan_block(*a, false).gy <= 65535u, "ValueError: too many chunks");
    return 0;
}

bool stride_ok(const dbk_blocknorm_args& a, const void* p, size_t ld) { return !p || a.n <= 1 || ld >= a.m; }

size_t block_work(const dbk_blocknorm_args& a) { return a.n && a.m ? (size_t)plan_block(a, true).gx * 5 * a.m * acc_size(a.dtype) : 0; }

}  // namespace
}  // namespace dbk

using namespace dbk;

extern "C" {

int dbk_blocknorm_args_size(void) { return (int)sizeof(dbk_blocknorm_args); }

int dbk_blocknorm(dbk_stream_t stream, const dbk_blocknorm_args* a)
{
    if (int rc = check_block(a)) return rc;
    const bool some = a->n && a->m;
    DBK_CHECK(!some || (a->O && (!a->next || a->Z)), "ValueError: null matrix");
    DBK_CHECK(stride_ok(*a, a->Y, a->ldy) && stride_ok(*a, a->R, a->ldr) && stride_ok(*a, a->gate, a->ldgate) && stride_ok(*a, a->O, a->ldo) && stride_ok(*a, a->Z, a->ldz),
              "ValueError: row strides must be at least the number of columns");
    if (!some) { clear_error(); return 0; }
    const block_plan p = plan_block(*a, false);
    hipStream_t st = as_stream(stream);
    with_row_type(a->dtype, [&](auto t) {
        typedef decltype(t) T;
        typedef typename acc_of<T>::type A;
        if (!block_layout<false>(p.lanes, a->group % row_vec<T>::N == 0, [&](auto lanes, auto exact) {
                k_block_fprop<T, lanes.value, exact.value><<<dim3(p.gx, p.gy), block_threads<lanes.value>(), 0, st>>>(
                    p.shape, (const T*)a->Y, (const T*)a->R, (const T*)a->gate, (const A*)a->gamma, (const A*)a->beta, (const A*)a->scale, (const A*)a->next_gamma,
                    (const A*)a->next_beta, (A)a->eps, (T*)a->O, (T*)a->Z, (A*)a->stats);
            })) {
            const size_t units = a->n * (a->m / a->group);
            k_block_fprop_wide<T><<<(unsigned)(units < WIDE_WGS ? units : WIDE_WGS), WIDE, 0, st>>>(
                p.shape, (const T*)a->Y, (const T*)a->R, (const T*)a->gate, (const A*)a->gamma, (const A*)a->beta, (const A*)a->scale, (const A*)a->next_gamma,
                (const A*)a->next_beta, (A)a->eps, (T*)a->O, a->next ? (T*)a->Z : nullptr, (A*)a->stats);
        }
    });
    DBK_LAUNCH_OK();
}

int dbk_blocknorm_bprop_workspace(const dbk_blocknorm_args* a, size_t* work_bytes)
{
    if (int rc = check_block(a)) return rc;
    DBK_CHECK(work_bytes, "ValueError: null result");
    *work_bytes = block_work(*a);
    clear_error();
    return 0;
}

int dbk_blocknorm_bprop(dbk_stream_t stream, const dbk_blocknorm_args* a, void* work, size_t work_bytes)
{
    if (int rc = check_block(a)) return rc;
    const bool some = a->n && a->m, weights = a->dgamma || a->dbeta || a->dscale || a->dnext_gamma || a->dnext_beta;
    DBK_CHECK(!some || (a->dY && (a->dR || a->next) && (!a->next || (a->O && a->dZ)) && (!(a->norm || a->next) || a->stats) && (!a->gate || a->dgate)), "ValueError: null matrix");
    DBK_CHECK(stride_ok(*a, a->Y, a->ldy) && stride_ok(*a, a->gate, a->ldgate) && stride_ok(*a, a->O, a->ldo) && stride_ok(*a, a->dR, a->lddr) && stride_ok(*a, a->dZ, a->lddz) &&
                  stride_ok(*a, a->dY, a->lddy) && stride_ok(*a, a->dR_in, a->lddr_in) && stride_ok(*a, a->dgate, a->lddgate),
              "ValueError: row strides must be at least the number of columns");
    const size_t need = weights ? block_work(*a) : 0;
    DBK_CHECK(!need || (work && work_bytes >= need), "ValueError: the workspace has %zu bytes, %zu are needed", work_bytes, need);
    hipStream_t st = as_stream(stream);
    const block_plan p = some ? plan_block(*a, true) : block_plan();
    if (some)
        with_row_type(a->dtype, [&](auto t) {
            typedef decltype(t) T;
            typedef typename acc_of<T>::type A;
            A* part = weights ? (A*)work : nullptr;
            if (!block_layout<true>(p.lanes, a->group % row_vec<T>::N == 0, [&](auto lanes, auto exact) {
                    auto kernel = a->rms ? k_block_bprop<T, lanes.value, exact.value, true> : k_block_bprop<T, lanes.value, exact.value, false>;
                    kernel<<<dim3(p.gx, p.gy), block_threads<lanes.value>(), 0, st>>>(
                        p.shape, (const T*)a->Y, (const T*)a->O, (const T*)a->gate, (const A*)a->gamma, (const A*)a->beta, (const A*)a->scale, (const A*)a->next_gamma,
                        (const A*)a->stats, (const T*)a->dR, (const T*)a->dZ, (T*)a->dY, (T*)a->dR_in, (T*)a->dgate, part);
                }))
                k_block_bprop_wide<T><<<p.gx, WIDE, 0, st>>>(p.shape, (const T*)a->Y, (const T*)a->O, (const T*)a->gate, (const A*)a->gamma, (const A*)a->beta, (const A*)a->scale,
                                                             (const A*)a->next_gamma, (const A*)a->stats, (const T*)a->dR, (const T*)a->dZ, (T*)a->dY, (T*)a->dR_in, (T*)a->dgate, part);
        });
    // (sums of no rows: zeros)
    if (weights) sum_partials(st, a->dtype, work, some ? p.gx : 0, {a->m, a->m, a->m, a->m, a->m}, {a->dgamma, a->dbeta, a->dscale, a->dnext_gamma, a->dnext_beta});
    DBK_LAUNCH_OK();
}

}  // extern "C"
