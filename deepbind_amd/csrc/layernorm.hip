// Layer norm of the rows of a matrix, or of every chunk of `group` consecutive columns of each row (the models' blocks of a
// row, as dbk_softmax takes them), forward and backward.
//
//   c = x - mean(x), r = 1 / sqrt(mean(c^2) + eps), h = c r, z = h gamma + beta
//   dx = r (q - mean(q) - h mean(q h)) with q = dz gamma,  dgamma = sum over rows of dz h,  dbeta = sum over rows of dz
//
// Bound by memory: the forward pass reads x and writes z, the backward pass reads x and dz and writes dx; a chunk's values stay
// in registers between the passes over them (mean, squares, result), so that each is read once. Measured: 130003 x 1440 bfloat16 forward
// 151 us (749 MB), backward 239 us (1.12 GB); 50021 rows of 64 chunks of 16 floats 79 and 140 us (410 and 615 MB). Chunks too wide for the registers are
// read three times either way, from the caches where they hold them: 5003 x 20001 floats 337 us forward, 900 both ways (0.8 and 1.6 GB).
#include <type_traits>
#include "rows_common.h"

namespace dbk {

// A chunk belongs to LANES neighbouring lanes (a power of two within a wave, or the 256 threads of a workgroup), each with NV
// vectors of 16 bytes, vector i at lane + i * LANES: consecutive lanes read consecutive memory. A workgroup holds CT chunks
// of a row side by side and RT = 256 / (LANES * CT) rows, and walks down the rows with its chunks' weights in registers.
struct norm_shape {
    unsigned n, nchunk, width, ct_log2, rstep;   // rows, chunks per row, columns per chunk, log2 of CT, rows per step of the grid
    size_t ldx, ldz;
};

template <int LANES, typename A> __device__ __forceinline__ A lanes_sum(A v, A* lds)
{
    constexpr int W = LANES < 64 ? LANES : 64;
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
    if constexpr (LANES > 64) {
        __syncthreads();                         // (the words may still be read from the sum before)
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = (lds[0] + lds[1]) + (lds[2] + lds[3]);
    }
    return v;
}

// two sums at once
template <int LANES, typename A> __device__ __forceinline__ void lanes_sum2(A& u, A& v, A* lds)
{
    constexpr int W = LANES < 64 ? LANES : 64;
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) {
        u += __shfl_xor(u, o);
        v += __shfl_xor(v, o);
    }
    if constexpr (LANES > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) { lds[threadIdx.x >> 6] = u; lds[4 + (threadIdx.x >> 6)] = v; }
        __syncthreads();
        u = (lds[0] + lds[1]) + (lds[2] + lds[3]);
        v = (lds[4] + lds[5]) + (lds[6] + lds[7]);
    }
}

// A chunk's mean and reciprocal deviation from its sum's mean `near`, the mean of the squared distances to that and the mean of the distances. The sum's
// roundings make `near` miss the mean by a few units in its last place, which is all there is where the values are equal, and more than their
// spread where they lie far from zero: the distances, of the spread's size, say by how much.
template <typename A> __device__ __forceinline__ void norm_stats(A near, A sq, A rest, A eps, A& mean, A& rstd)
{
    const A var = fma(-rest, rest, sq);
    mean = near + rest;
    rstd = A(1) / sqrt((var < A(0) ? A(0) : var) + eps);        // (a NaN stays)
}

// A row's values come while the row before it is worked on, and stay as they lie in memory: for bfloat16 half the registers of what is
// computed from them, which is computed twice instead.
template <typename T, int LANES, int NV, bool EXACT>
__global__ __launch_bounds__(256) void k_norm_fprop(norm_shape p, const T* __restrict__ X, const typename acc_of<T>::type* __restrict__ gamma,
                                                    const typename acc_of<T>::type* __restrict__ beta, typename acc_of<T>::type eps,
                                                    T* __restrict__ Z, typename acc_of<T>::type* __restrict__ stats)
{
    typedef typename acc_of<T>::type A;
    constexpr int V = row_vec<T>::N;
    __shared__ A lds[8];
    const unsigned unit = threadIdx.x / LANES, lane = threadIdx.x % LANES;
    const unsigned chunk = (blockIdx.y << p.ct_log2) + (unit & ((1u << p.ct_log2) - 1u));
    const unsigned first = blockIdx.x * (256u / LANES) >> p.ct_log2;
    const bool own = chunk < p.nchunk;
    A g[NV][V], b[NV][V];
    unsigned valid[NV];
    const A inv = A(1) / (A)p.width;
    const size_t column = (size_t)chunk * p.width + lane * V;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const unsigned c = (lane + i * LANES) * V;
        valid[i] = own && c < p.width ? p.width - c : 0u;
        load_weights(g[i], gamma ? gamma + column + i * LANES * V : nullptr, valid[i], A(1));
        load_weights(b[i], beta ? beta + column + i * LANES * V : nullptr, valid[i], A(0));
    }
    unsigned row = first + (unit >> p.ct_log2);
    raw_vec<T, EXACT> next[NV];
    auto fetch = [&]() {
        const T* x = X + (size_t)row * p.ldx + column;
#pragma unroll
        for (int i = 0; i < NV; ++i) next[i].load(x + i * LANES * V, row < p.n ? valid[i] : 0u);
    };
    fetch();
    // (every lane of a workgroup makes the same number of steps: the sums of LANES = 256 meet at barriers)
    for (unsigned left = first; left < p.n; left += p.rstep) {
        raw_vec<T, EXACT> x[NV];
        const unsigned now = row;
        A sum = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            x[i] = next[i];
#pragma unroll
            for (int j = 0; j < V; ++j) sum += x[i][j];
        }
        row += p.rstep;
        fetch();
        const A near = lanes_sum<LANES>(sum, lds) * inv;
        A sq = 0, rest = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const A c = (EXACT ? valid[i] != 0 : j < (int)valid[i]) ? x[i][j] - near : A(0);
                sq = fma(c, c, sq);
                rest += c;
            }
        lanes_sum2<LANES>(sq, rest, lds);
        A mean, rstd;
        norm_stats(near, sq * inv, rest * inv, eps, mean, rstd);
        if (now >= p.n) continue;
        T* z = Z + (size_t)now * p.ldz + column;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            row_vec<T> o;
            x[i].forget();
#pragma unroll
            for (int j = 0; j < V; ++j) o.v[j] = fma((x[i][j] - mean) * rstd, g[i][j], b[i][j]);
            store_vec<EXACT>(o, z + i * LANES * V, valid[i]);
        }
        if (stats && own && lane == 0) {
            const size_t at = (size_t)now * p.nchunk + chunk;
            stats[at] = mean;
            stats[(size_t)p.n * p.nchunk + at] = rstd;
        }
    }
}

// The backward pass walks the rows the same way and adds dz h and dz up in registers; the workgroup's row lanes are added in
// LDS at the end, in a fixed order, and leave one row of partial sums per workgroup: part[blockIdx.x][2][nchunk * width].
// (Lanes without a column hold dz = 0, which leaves nothing in any sum.)
template <typename T, int LANES, int NV, bool EXACT>
__global__ __launch_bounds__(256) void k_norm_bprop(norm_shape p, size_t lddz, const T* __restrict__ X, const typename acc_of<T>::type* __restrict__ gamma,
                                                    const typename acc_of<T>::type* __restrict__ stats, const T* __restrict__ dZ,
                                                    T* __restrict__ dX, typename acc_of<T>::type* __restrict__ part)
{
    typedef typename acc_of<T>::type A;
    constexpr int V = row_vec<T>::N;
    __shared__ A lds[8];
    __shared__ A rows_lds[2][256][V + 1];
    const unsigned unit = threadIdx.x / LANES, lane = threadIdx.x % LANES;
    const unsigned chunk = (blockIdx.y << p.ct_log2) + (unit & ((1u << p.ct_log2) - 1u));
    const unsigned first = blockIdx.x * (256u / LANES) >> p.ct_log2;
    const bool own = chunk < p.nchunk;
    A g[NV][V], dg[NV][V], db[NV][V];
    unsigned valid[NV];
    const A inv = A(1) / (A)p.width;
    const size_t column = (size_t)chunk * p.width + lane * V;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const unsigned c = (lane + i * LANES) * V;
        valid[i] = own && c < p.width ? p.width - c : 0u;
        load_weights(g[i], gamma ? gamma + column + i * LANES * V : nullptr, valid[i], A(1));
#pragma unroll
        for (int j = 0; j < V; ++j) dg[i][j] = db[i][j] = A(0);
    }
    unsigned row = first + (unit >> p.ct_log2);
    raw_vec<T, EXACT> nx[NV], nd[NV];
    A nmean = 0, nrstd = 0;
    auto fetch = [&]() {
        const bool here = own && row < p.n;
        const T *x = X + (size_t)row * p.ldx + column, *d = dZ + (size_t)row * lddz + column;
        const size_t at = (size_t)row * p.nchunk + chunk;
        nmean = here ? stats[at] : A(0);
        nrstd = here ? stats[(size_t)p.n * p.nchunk + at] : A(0);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            nx[i].load(x + i * LANES * V, here ? valid[i] : 0u);
            nd[i].load(d + i * LANES * V, here ? valid[i] : 0u);
        }
    };
    fetch();
    for (unsigned left = first; left < p.n; left += p.rstep) {
        raw_vec<T, EXACT> x[NV], d[NV];
        const A mean = nmean, rstd = nrstd;
        const unsigned now = row;
        A s1 = 0, s2 = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) { x[i] = nx[i]; d[i] = nd[i]; }
        row += p.rstep;
        fetch();
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const A h = (x[i][j] - mean) * rstd, q = d[i][j] * g[i][j];
                dg[i][j] = fma(d[i][j], h, dg[i][j]);
                db[i][j] += d[i][j];
                s1 += q;
                s2 = fma(q, h, s2);
            }
        lanes_sum2<LANES>(s1, s2, lds);
        s1 *= inv;
        s2 *= inv;
        if (!own || now >= p.n) continue;
        T* dx = dX + (size_t)now * p.ldz + column;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            row_vec<T> o;
            x[i].forget();
            d[i].forget();
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const A h = (x[i][j] - mean) * rstd;
                o.v[j] = rstd * (fma(d[i][j], g[i][j], -s1) - h * s2);
            }
            store_vec<EXACT>(o, dx + i * LANES * V, valid[i]);
        }
    }
    if (!part) return;
    const unsigned across = LANES << p.ct_log2;                 // threads of one row lane
    const size_t m = (size_t)p.nchunk * p.width;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < V; ++j) { rows_lds[0][threadIdx.x][j] = dg[i][j]; rows_lds[1][threadIdx.x][j] = db[i][j]; }
        sum_strips(rows_lds[0], across, V);
        sum_strips(rows_lds[1], across, V);
        if (threadIdx.x >= across || !valid[i]) continue;
        const unsigned c = (lane + i * LANES) * V;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (j >= (int)valid[i]) continue;
            A* o = part + (size_t)blockIdx.x * 2u * m + (size_t)chunk * p.width + c + j;
            o[0] = rows_lds[0][threadIdx.x][j];
            o[m] = rows_lds[1][threadIdx.x][j];
        }
    }
}

// Chunks too wide for the registers of 256 threads: a workgroup per chunk reads it once per pass (from the caches after the first).
template <typename T>
__global__ __launch_bounds__(256) void k_norm_fprop_wide(norm_shape p, const T* __restrict__ X, const typename acc_of<T>::type* __restrict__ gamma,
                                                         const typename acc_of<T>::type* __restrict__ beta, typename acc_of<T>::type eps,
                                                         T* __restrict__ Z, typename acc_of<T>::type* __restrict__ stats)
{
    typedef typename acc_of<T>::type A;
    constexpr int V = row_vec<T>::N;
    __shared__ A lds[8];
    const A inv = A(1) / (A)p.width;
    for (size_t u = blockIdx.x; u < (size_t)p.n * p.nchunk; u += gridDim.x) {
        const size_t row = u / p.nchunk, chunk = u % p.nchunk;
        const T* x = X + row * p.ldx + chunk * p.width;
        T* z = Z + row * p.ldz + chunk * p.width;
        A s = 0;
        row_vec<T> v;
        for (unsigned c = threadIdx.x * V; c < p.width; c += 256u * V) {
            v.load(x + c, p.width - c);
#pragma unroll
            for (int j = 0; j < V; ++j) s += v.v[j];
        }
        const A near = lanes_sum<256>(s, lds) * inv;
        A rest = s = 0;
        for (unsigned c = threadIdx.x * V; c < p.width; c += 256u * V) {
            v.load(x + c, p.width - c);
#pragma unroll
            for (int j = 0; j < V; ++j) { const A d = c + j < p.width ? v.v[j] - near : A(0); s += d * d; rest += d; }
        }
        lanes_sum2<256>(s, rest, lds);
        A mean, rstd;
        norm_stats(near, s * inv, rest * inv, eps, mean, rstd);
        for (unsigned c = threadIdx.x * V; c < p.width; c += 256u * V) {
            A g[V], b[V];
            v.load(x + c, p.width - c);
            load_weights(g, gamma ? gamma + chunk * p.width + c : nullptr, p.width - c, A(1));
            load_weights(b, beta ? beta + chunk * p.width + c : nullptr, p.width - c, A(0));
#pragma unroll
            for (int j = 0; j < V; ++j) v.v[j] = (v.v[j] - mean) * rstd * g[j] + b[j];
            v.store(z + c, p.width - c);
        }
        if (stats && threadIdx.x == 0) { stats[u] = mean; stats[(size_t)p.n * p.nchunk + u] = rstd; }
    }
}

template <typename T>
__global__ __launch_bounds__(256) void k_norm_bprop_wide(norm_shape p, size_t lddz, const T* __restrict__ X, const typename acc_of<T>::type* __restrict__ gamma,
                                                         const typename acc_of<T>::type* __restrict__ stats, const T* __restrict__ dZ, T* __restrict__ dX)
{
    typedef typename acc_of<T>::type A;
    constexpr int V = row_vec<T>::N;
    __shared__ A lds[4];
    const A inv = A(1) / (A)p.width;
    for (size_t u = blockIdx.x; u < (size_t)p.n * p.nchunk; u += gridDim.x) {
        const size_t row = u / p.nchunk, chunk = u % p.nchunk;
        const T *x = X + row * p.ldx + chunk * p.width, *dz = dZ + row * lddz + chunk * p.width;
        T* dx = dX + row * p.ldz + chunk * p.width;
        const A mean = stats[u], rstd = stats[(size_t)p.n * p.nchunk + u];
        A s1 = 0, s2 = 0, g[V];
        row_vec<T> v, d;
        for (unsigned c = threadIdx.x * V; c < p.width; c += 256u * V) {
            v.load(x + c, p.width - c);
            d.load(dz + c, p.width - c);
            load_weights(g, gamma ? gamma + chunk * p.width + c : nullptr, p.width - c, A(1));
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const A q = d.v[j] * g[j];
                s1 += q;
                s2 += c + j < p.width ? q * ((v.v[j] - mean) * rstd) : A(0);
            }
        }
        s1 = lanes_sum<256>(s1, lds) * inv;
        s2 = lanes_sum<256>(s2, lds) * inv;
        for (unsigned c = threadIdx.x * V; c < p.width; c += 256u * V) {
            v.load(x + c, p.width - c);
            d.load(dz + c, p.width - c);
            load_weights(g, gamma ? gamma + chunk * p.width + c : nullptr, p.width - c, A(1));
#pragma unroll
            for (int j = 0; j < V; ++j) d.v[j] = rstd * (d.v[j] * g[j] - s1 - (v.v[j] - mean) * rstd * s2);
            d.store(dx + c, p.width - c);
        }
    }
}

// Their weights' gradient: a thread per vector of columns of one chunk, down the rows of its workgroup.
template <typename T>
__global__ __launch_bounds__(256) void k_norm_wgrad_wide(norm_shape p, size_t lddz, const T* __restrict__ X, const typename acc_of<T>::type* __restrict__ stats,
                                                         const T* __restrict__ dZ, typename acc_of<T>::type* __restrict__ part)
{
    typedef typename acc_of<T>::type A;
    constexpr int V = row_vec<T>::N;
    const unsigned chunk = blockIdx.z, c = (blockIdx.y * 256u + threadIdx.x) * V;
    if (c >= p.width) return;
    const unsigned valid = p.width - c;
    A dg[V], db[V];
#pragma unroll
    for (int j = 0; j < V; ++j) dg[j] = db[j] = A(0);
    for (size_t row = blockIdx.x; row < p.n; row += gridDim.x) {
        row_vec<T> v, d;
        v.load(X + row * p.ldx + (size_t)chunk * p.width + c, valid);
        d.load(dZ + row * lddz + (size_t)chunk * p.width + c, valid);
        const size_t at = row * p.nchunk + chunk;
        const A mean = stats[at], rstd = stats[(size_t)p.n * p.nchunk + at];
#pragma unroll
        for (int j = 0; j < V; ++j) { dg[j] += d.v[j] * ((v.v[j] - mean) * rstd); db[j] += d.v[j]; }
    }
    const size_t m = (size_t)p.nchunk * p.width;
    A* o = part + (size_t)blockIdx.x * 2u * m + (size_t)chunk * p.width + c;
#pragma unroll
    for (int j = 0; j < V; ++j) if (j < (int)valid) { o[j] = dg[j]; o[m + j] = db[j]; }
}

// out[c] = sum over units of part[unit][c] in a fixed order: 16 columns x 64 groups of units per workgroup, each thread its
// group's units one after another, the groups' sums through LDS.
template <typename A>
__global__ __launch_bounds__(1024) void k_sum_partials(const A* __restrict__ part, size_t units, size_t first, size_t ncol, size_t n0, A* out0, size_t n1, A* out1, A* out2)
{
    __shared__ A lds[64][17];
    const unsigned x = threadIdx.x & 15u, y = threadIdx.x >> 4;
    const size_t c = first + (size_t)blockIdx.x * 16u + x;
    A s = 0;
    if (c < ncol)
#pragma unroll 8
        for (size_t u = y; u < units; u += 64u) s += part[u * ncol + c];
    lds[y][x] = s;
    __syncthreads();
    for (unsigned o = 32; o > 0; o >>= 1) {
        if (y < o) lds[y][x] += lds[y + o][x];
        __syncthreads();
    }
    if (y == 0 && c < ncol) {
        A* out = c < n0 ? out0 : c < n0 + n1 ? out1 : out2;
        if (out) out[c < n0 ? c : c < n0 + n1 ? c - n0 : c - n0 - n1] = lds[0][x];
    }
}

int sum_partials(hipStream_t st, int dtype, const void* part, size_t units, size_t n0, void* out0, size_t n1, void* out1, size_t n2, void* out2)
{
    const size_t ncol = n0 + n1 + n2;
    constexpr size_t MOST = size_t(1) << 25;     // columns of a launch (grid_fits)
    for (size_t first = 0; first < ncol; first += MOST) {
        const unsigned wgs = divup(ncol - first < MOST ? ncol - first : MOST, 16);
        if (dtype == DBK_F64)
            k_sum_partials<double><<<wgs, 1024, 0, st>>>((const double*)part, units, first, ncol, n0, (double*)out0, n1, (double*)out1, (double*)out2);
        else
            k_sum_partials<float><<<wgs, 1024, 0, st>>>((const float*)part, units, first, ncol, n0, (float*)out0, n1, (float*)out1, (float*)out2);
    }
    return 0;
}

namespace {

// How a call is laid out: lanes and vectors per chunk, chunks side by side, workgroups down the rows.
struct norm_plan {
    int lanes, nv;                               // lanes == 0: the wide kernels
    unsigned ct_log2, gx, gy;
    norm_shape shape;
};

constexpr unsigned NORM_WGS = 2048;              // workgroups that walk the rows: eight per CU
constexpr int NORM_NV_BLOCK = 4;                 // vectors per thread of the 256-thread form: 16 registers (float) per array

norm_plan plan_norm(int dtype, size_t n, size_t m, size_t group)
{
    norm_plan p;
    const size_t vecs = (group + 16 / row_size(dtype) - 1) / (16 / row_size(dtype)), nchunk = m / group;
    p.lanes = 64;
    p.nv = 1;
    if (vecs <= 64) { p.lanes = 1; while ((size_t)p.lanes < vecs) p.lanes *= 2; }
    else if (vecs <= 256) p.nv = (int)((vecs + 63) / 64);
    else if (vecs <= 256 * NORM_NV_BLOCK) { p.lanes = 256; p.nv = vecs <= 512 ? 2 : NORM_NV_BLOCK; }
    else p.lanes = 0;
    // Chunks side by side: the power of two that costs least, counting the lanes whose chunk does not exist and, against short pieces of
    // rows, 128 bytes more for every piece.
    unsigned best = 0;
    double least = 1e300;
    for (unsigned c = 0; p.lanes && (unsigned)p.lanes << c <= 256u; ++c) {
        const size_t tiles = (nchunk + (size_t(1) << c) - 1) >> c;
        const double cost = (double)(tiles << c) * (1.0 + 128.0 / (double)((size_t)p.lanes * 16 << c));
        if (cost <= least) { least = cost; best = c; }
        if (tiles == 1) break;
    }
    p.ct_log2 = best;
    const unsigned rt = p.lanes ? (256u / p.lanes) >> best : 1u;
    p.gy = p.lanes ? divup(nchunk, size_t(1) << best) : 1u;
    const unsigned wgs = p.nv > 1 ? NORM_WGS / 2 : NORM_WGS, most = wgs / p.gy ? wgs / p.gy : 1u;      // (several vectors: two waves per SIMD fit)
    p.gx = divup(n, rt);
    if (p.gx > most) p.gx = most;
    p.shape.n = (unsigned)n;
    p.shape.nchunk = (unsigned)nchunk;
    p.shape.width = (unsigned)group;
    p.shape.ct_log2 = best;
    p.shape.rstep = p.gx * rt;
    return p;
}

constexpr unsigned WIDE_ROWS = 256;              // workgroups down the rows of the wide form's weight gradient

template <typename F> bool norm_layout(int lanes, int nv, bool exact, F f)
{
#define DBK_NORM_CASE(L, V)                                                                              \
    if (lanes == L && nv == V) {                                                                         \
        if (exact) f(std::integral_constant<int, L>(), std::integral_constant<int, V>(), std::true_type());      \
        else f(std::integral_constant<int, L>(), std::integral_constant<int, V>(), std::false_type());           \
        return true;                                                                                     \
    }
    DBK_NORM_CASE(1, 1) DBK_NORM_CASE(2, 1) DBK_NORM_CASE(4, 1) DBK_NORM_CASE(8, 1) DBK_NORM_CASE(16, 1) DBK_NORM_CASE(32, 1)
    DBK_NORM_CASE(64, 1) DBK_NORM_CASE(64, 2) DBK_NORM_CASE(64, 3) DBK_NORM_CASE(64, 4) DBK_NORM_CASE(256, 2) DBK_NORM_CASE(256, 4)
#undef DBK_NORM_CASE
    return false;
}

int check_norm(int dtype, const void* X, size_t ldx, size_t n, size_t m, size_t group, const void* Z, size_t ldz)
{
    DBK_ROW_DTYPE_OK(dtype);
    DBK_CHECK(group >= 1 && m % group == 0, "ValueError: the number of columns must be divisible by the chunk's");
    DBK_CHECK(n < (size_t(1) << 31) && m < (size_t(1) << 31), "ValueError: matrix too large (%zu x %zu)", n, m);
    DBK_CHECK(plan_norm(dtype, 1, m, group).gy <= 65535u && (plan_norm(dtype, 1, m, group).lanes || m / group <= 65535u), "ValueError: too many chunks");
    DBK_CHECK(n == 0 || (X && Z), "ValueError: null matrix");
    DBK_CHECK(n <= 1 || (ldx >= m && ldz >= m), "ValueError: row strides must be at least the number of columns");
    return 0;
}

}  // namespace
}  // namespace dbk

using namespace dbk;

extern "C" {

int dbk_layernorm(dbk_stream_t stream, int dtype, const void* X, size_t ldx, const void* gamma, const void* beta, size_t n, size_t m, size_t group,
                  double eps, void* Z, size_t ldz, void* stats)
{
    if (n && !m) n = 0;
    if (int rc = check_norm(dtype, X, ldx, n, m, group, Z, ldz)) return rc;
    if (!n) { clear_error(); return 0; }
    norm_plan p = plan_norm(dtype, n, m, group);
    p.shape.ldx = ldx;
    p.shape.ldz = ldz;
    hipStream_t st = as_stream(stream);
    with_row_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        typedef typename acc_of<T>::type A;
        if (!norm_layout(p.lanes, p.nv, group % row_vec<T>::N == 0, [&](auto lanes, auto nv, auto exact) {
                k_norm_fprop<T, lanes.value, nv.value, exact.value><<<dim3(p.gx, p.gy), 256, 0, st>>>(p.shape, (const T*)X, (const A*)gamma, (const A*)beta, (A)eps, (T*)Z, (A*)stats);
            })) {
            const size_t units = n * (m / group);
            k_norm_fprop_wide<T><<<(unsigned)(units < NORM_WGS ? units : NORM_WGS), 256, 0, st>>>(p.shape, (const T*)X, (const A*)gamma, (const A*)beta, (A)eps, (T*)Z, (A*)stats);
        }
    });
    DBK_LAUNCH_OK();
}

int dbk_layernorm_bprop_workspace(int dtype, size_t n, size_t m, size_t group, size_t* work_bytes)
{
    DBK_ROW_DTYPE_OK(dtype);
    DBK_CHECK(work_bytes, "ValueError: null result");
    DBK_CHECK(group >= 1 && m % group == 0, "ValueError: the number of columns must be divisible by the chunk's");
    *work_bytes = 0;
    if (n && m) {
        const norm_plan p = plan_norm(dtype, n, m, group);
        *work_bytes = (p.lanes ? p.gx : n < WIDE_ROWS ? n : WIDE_ROWS) * 2 * m * acc_size(dtype);
    }
    clear_error();
    return 0;
}

int dbk_layernorm_bprop(dbk_stream_t stream, int dtype, const void* X, size_t ldx, const void* gamma, const void* stats, const void* dZ, size_t lddz,
                        size_t n, size_t m, size_t group, void* dX, size_t lddx, void* dgamma, void* dbeta, void* work, size_t work_bytes)
{
    const size_t rows = n;
    if (n && !m) n = 0;
    if (int rc = check_norm(dtype, X, ldx, n, m, group, dX, lddx)) return rc;
    DBK_CHECK(n == 0 || (stats && dZ), "ValueError: null matrix");
    DBK_CHECK(n <= 1 || lddz >= m, "ValueError: row strides must be at least the number of columns");
    const bool weights = dgamma || dbeta;
    const size_t per_wg = 256 * (dtype == DBK_F64 ? 2 : dtype == DBK_BF16 ? 8 : 4);       // columns of a workgroup of the wide form
    DBK_CHECK(!weights || !n || plan_norm(dtype, n, m, group).lanes || grid_fits(1, 256, (group + per_wg - 1) / per_wg), "ValueError: chunks too wide (%zu columns)", group);
    size_t need = 0;
    if (weights) if (int rc = dbk_layernorm_bprop_workspace(dtype, rows, m, group, &need)) return rc;
    DBK_CHECK(!need || (work && work_bytes >= need), "ValueError: the workspace has %zu bytes, %zu are needed", work_bytes, need);
    hipStream_t st = as_stream(stream);
    if (!n) {
        sum_partials(st, dtype, nullptr, 0, m, dgamma, m, dbeta, 0, nullptr);         // (sums of no rows: zeros)
        DBK_LAUNCH_OK();
    }
    norm_plan p = plan_norm(dtype, n, m, group);
    p.shape.ldx = ldx;
    p.shape.ldz = lddx;
    size_t units = p.gx;
    with_row_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        typedef typename acc_of<T>::type A;
        A* part = weights ? (A*)work : nullptr;
        if (!norm_layout(p.lanes, p.nv, group % row_vec<T>::N == 0, [&](auto lanes, auto nv, auto exact) {
                k_norm_bprop<T, lanes.value, nv.value, exact.value><<<dim3(p.gx, p.gy), 256, 0, st>>>(p.shape, lddz, (const T*)X, (const A*)gamma, (const A*)stats, (const T*)dZ, (T*)dX, part);
            })) {
            const size_t chunks = n * (m / group);
            k_norm_bprop_wide<T><<<(unsigned)(chunks < NORM_WGS ? chunks : NORM_WGS), 256, 0, st>>>(p.shape, lddz, (const T*)X, (const A*)gamma, (const A*)stats, (const T*)dZ, (T*)dX);
            units = n < WIDE_ROWS ? n : WIDE_ROWS;
            if (weights)
                k_norm_wgrad_wide<T><<<dim3((unsigned)units, divup(group, 256 * row_vec<T>::N), (unsigned)(m / group)), 256, 0, st>>>(p.shape, lddz, (const T*)X, (const A*)stats,
                                                                                                                                (const T*)dZ, part);
        }
    });
    if (weights) sum_partials(st, dtype, work, units, m, dgamma, m, dbeta, 0, nullptr);
    DBK_LAUNCH_OK();
}

}  // extern "C"
