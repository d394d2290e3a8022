// Causal convolution of up to four taps along the rows of every region of a map, a filter per channel:
//
//   p[t] = b + sum_j W[j] x[t - K + 1 + j]  (rows before the region's first: the given state, or zeros),  z = p sigmoid(p), or p
//   dp = dz sigmoid(p) (1 + p (1 - sigmoid(p))),  dx[t] = sum_j W[j] dp[t + K - 1 - j],  dW[j] = sum_t dp[t] x[t - K + 1 + j],  db = sum_t dp[t]
//
// Bound by memory: x in and z out forward, x and dz in and dx out backward (p is formed again from x: reading it would cost a
// third map, keeping it another). A lane owns four channels (two of double) and walks down a strip of rows with the last K - 1 of
// them in registers, so that a row is read once but for the K - 1 rows above each strip, which the caches hold. Measured: 106 502
// rows of 1024 bfloat16 83 us forward and 152 us backward (436 and 654 MB), 193 495 rows of 256 floats 81 us (396 MB).
#include <type_traits>
#include "rows_common.h"

namespace dbk {

// Four channels per lane: 16 bytes of float. (Eight bfloat16 would be 16 bytes too, but the weights, their sums and the last rows of eight
// channels take twice the registers, and fewer waves then keep memory busy.)
template <typename T> using conv_vec = row_vec<T, sizeof(T) == 8 ? 2 : 4>;

struct conv_shape {
    unsigned N, D, nregion, seg;                 // rows, channels, regions, rows per segment of a long region
    unsigned ct_log2, silu;                      // log2 of the lanes side by side; activation
    size_t ldx, ldz;
};

template <typename T, int K> struct conv_weights {
    typedef typename acc_of<T>::type A;
    static constexpr int V = conv_vec<T>::N;
    A w[K][V], b[V];
    __device__ __forceinline__ void load(const A* W, const A* bias, unsigned D, unsigned c, unsigned valid)
    {
#pragma unroll
        for (int j = 0; j < K; ++j) load_weights(w[j], W + (size_t)j * D + c, valid, A(0));
        load_weights(b, bias ? bias + c : nullptr, valid, A(0));
    }
};

// row t of region r (t may lie up to K - 1 rows before its start)
template <typename T, int K>
__device__ __forceinline__ void conv_row(conv_vec<T>& v, const T* X, size_t ldx, const T* state, unsigned D, unsigned c, unsigned valid,
                                         unsigned r, row_range g, int64_t t)
{
    if (t >= (int64_t)g.start) v.load(X + (size_t)t * ldx + c, valid);
    else if (state) v.load(state + ((size_t)r * (K - 1) + (size_t)(t - g.start + K - 1)) * D + c, valid);
    else v.fill(typename acc_of<T>::type(0));
}

constexpr int CONV_AHEAD = 4;                    // rows that are fetched together, while the four before them are worked on
// the next CONV_AHEAD rows from `p` on, the last of `left` rows again behind it
template <typename T, bool EXACT> struct conv_ahead {
    raw_vec<T, EXACT, conv_vec<T>::N> v[CONV_AHEAD];
    __device__ __forceinline__ void fetch(const T*& p, size_t ld, unsigned valid, int64_t left)
    {
#pragma unroll
        for (int i = 0; i < CONV_AHEAD; ++i) {
            v[i].load(p, valid);
            p += i + 1 < left ? ld : 0;
        }
    }
    __device__ __forceinline__ void to(conv_vec<T>& x, int i) const
    {
#pragma unroll
        for (int j = 0; j < conv_vec<T>::N; ++j) x.v[j] = v[i][j];
    }
};

template <typename T, int K, bool EXACT>
__device__ __forceinline__ void conv_strip(conv_shape p, const conv_weights<T, K>& w, const T* X, const T* state, T* Z, unsigned c, unsigned valid,
                                           unsigned r, row_range g, unsigned from, unsigned to)
{
    typedef typename acc_of<T>::type A;
    constexpr int V = conv_vec<T>::N, U = CONV_AHEAD;
    if (from >= to || !valid) return;
    conv_vec<T> x[K - 1 + U];
    conv_ahead<T, EXACT> next;
    const T* xp = X + (size_t)from * p.ldx + c;
    T* zp = Z + (size_t)from * p.ldz + c;
    next.fetch(xp, p.ldx, valid, to - from);
#pragma unroll
    for (int j = 0; j < K - 1; ++j) conv_row<T, K>(x[j], X, p.ldx, state, p.D, c, valid, r, g, (int64_t)from - (K - 1) + j);
    for (unsigned t = from; t < to; t += U) {
#pragma unroll
        for (int i = 0; i < U; ++i) next.to(x[K - 1 + i], i);
        if (to - t > (unsigned)U) next.fetch(xp, p.ldx, valid, to - t - U);
#pragma unroll
        for (int i = 0; i < U; ++i) {
            if (t + i >= to) break;
            conv_vec<T> z;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                A a = w.b[v];
#pragma unroll
                for (int j = 0; j < K; ++j) a = fma(w.w[j][v], x[i + j].v[v], a);
                z.v[v] = p.silu ? a * sigmoid_of(a) : a;
            }
            store_vec<EXACT>(z, zp, valid);
            zp += p.ldz;
        }
#pragma unroll
        for (int j = 0; j < K - 1; ++j) x[j] = x[U + j];
    }
}

// A workgroup's lanes are 2^ct_log2 vectors of channels by strips of rows. Item i < nregion is the first segment of region i (all of it, mostly),
// the items behind are the slots of the other segments.
struct conv_item { unsigned r, from, len; row_range g; };
__device__ __forceinline__ bool conv_item_at(const conv_shape& p, const uint32_t* regions, const uint32_t* marks, unsigned i, conv_item& s)
{
    unsigned k = 0;
    if (i < p.nregion) {
        s.r = i;
        s.g = region_rows(regions, i, p.N);
    } else if (!slot_segment(regions, p.nregion, p.N, marks, i - p.nregion, p.seg, s.r, s.g, k))
        return false;
    s.from = s.g.start + k * p.seg;
    s.len = min(s.g.end - s.from, p.seg);
    return true;
}

__global__ __launch_bounds__(256) void k_conv_mark(conv_shape p, const uint32_t* __restrict__ regions, uint32_t* __restrict__ marks)
{
    const unsigned r = blockIdx.x * 4u + (threadIdx.x >> 6);
    if (r < p.nregion) mark_segments(marks, r, region_rows(regions, r, p.N), p.seg, threadIdx.x & 63u, 64u);
}

template <typename T, int K, bool EXACT>
__global__ __launch_bounds__(256) void k_conv_fprop(conv_shape p, const T* __restrict__ X, const typename acc_of<T>::type* __restrict__ W,
                                                    const typename acc_of<T>::type* __restrict__ bias, const uint32_t* __restrict__ regions,
                                                    const uint32_t* __restrict__ marks, const T* __restrict__ state, T* __restrict__ Z, T* __restrict__ last)
{
    constexpr int V = conv_vec<T>::N;
    conv_item s;
    if (!conv_item_at(p, regions, marks, blockIdx.x, s)) return;
    const unsigned x = threadIdx.x & ((1u << p.ct_log2) - 1u), y = threadIdx.x >> p.ct_log2, strips = 256u >> p.ct_log2;
    const unsigned c = ((blockIdx.y << p.ct_log2) + x) * V, valid = c < p.D ? p.D - c : 0u;
    conv_weights<T, K> w;
    w.load(W, bias, p.D, c, valid);
    const unsigned strip = (s.len + strips - 1) / strips;
    conv_strip<T, K, EXACT>(p, w, X, state, Z, c, valid, s.r, s.g, s.from + min(y * strip, s.len), s.from + min((y + 1) * strip, s.len));
    if (last && blockIdx.x < p.nregion && y < K - 1 && valid) {          // the K - 1 rows that the next piece of this sequence needs
        conv_vec<T> v;
        conv_row<T, K>(v, X, p.ldx, state, p.D, c, valid, s.r, s.g, (int64_t)s.g.end - (K - 1) + y);
        v.store(last + ((size_t)s.r * (K - 1) + y) * p.D + c, valid);
    }
}

// Backward of rows [from, to) of region g, adding to the lane's dW, db. Each row's dp is formed once, but for the K - 1 rows below
// the strip that its own last dx need.
template <typename T, int K> struct conv_sums {
    typedef typename acc_of<T>::type A;
    static constexpr int V = conv_vec<T>::N;
    A dw[K][V], db[V];
    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            db[v] = A(0);
#pragma unroll
            for (int j = 0; j < K; ++j) dw[j][v] = A(0);
        }
    }
};
template <typename T, int K, bool EXACT>
__device__ __forceinline__ void conv_strip_bprop(conv_shape p, size_t lddz, const conv_weights<T, K>& w, conv_sums<T, K>& sums, const T* X, const T* dZ, T* dX,
                                                 unsigned c, unsigned valid, row_range g, unsigned from, unsigned to)
{
    typedef typename acc_of<T>::type A;
    constexpr int V = conv_vec<T>::N, U = CONV_AHEAD;
    if (from >= to || !valid) return;
    conv_vec<T> x[K - 1 + U], dp[K];             // rows t - K + 1 on; dp[j] = dp of row t - K + 1 + j
    conv_ahead<T, EXACT> nx, nd;
    const T *xp = X + (size_t)from * p.ldx + c, *dp_ = dZ + (size_t)from * lddz + c;
    T* op = dX + (size_t)from * p.ldz + c;
    // rows of the region from `from` on, rows of the strip, and rows walked: K - 1 more, whose dp the strip's last rows need
    const int64_t rows = (int64_t)g.end - from, own = to - from, stop = own + (K - 1);
    nx.fetch(xp, p.ldx, valid, rows);
    nd.fetch(dp_, lddz, valid, rows);
#pragma unroll
    for (int j = 0; j < K; ++j) dp[j].fill(A(0));
#pragma unroll
    for (int j = 0; j < K - 1; ++j) conv_row<T, K>(x[j], X, p.ldx, (const T*)nullptr, p.D, c, valid, 0u, g, (int64_t)from - (K - 1) + j);
    for (int64_t t0 = 0; t0 < stop; t0 += U) {
        conv_vec<T> d[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            nx.to(x[K - 1 + i], i);
            nd.to(d[i], i);
        }
        if (t0 + U < stop) {
            nx.fetch(xp, p.ldx, valid, rows - t0 - U);
            nd.fetch(dp_, lddz, valid, rows - t0 - U);
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int64_t t = t0 + i;
            if (t >= stop) break;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                A dpre = d[i].v[v];
                if (p.silu) {
                    A a = w.b[v];
#pragma unroll
                    for (int j = 0; j < K; ++j) a = fma(w.w[j][v], x[i + j].v[v], a);
                    const A s = sigmoid_of(a);
                    dpre *= s * fma(a, A(1) - s, A(1));
                }
                dp[K - 1].v[v] = t < rows ? dpre : A(0);         // (behind the region nothing is sent back)
            }
            if (t < own) {
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    sums.db[v] += dp[K - 1].v[v];
#pragma unroll
                    for (int j = 0; j < K; ++j) sums.dw[j][v] = fma(dp[K - 1].v[v], x[i + j].v[v], sums.dw[j][v]);
                }
            }
            if (t >= K - 1) {
                conv_vec<T> o;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    A a = 0;
#pragma unroll
                    for (int j = 0; j < K; ++j) a = fma(w.w[j][v], dp[K - 1 - j].v[v], a);
                    o.v[v] = a;
                }
                store_vec<EXACT>(o, op, valid);
                op += p.ldz;
            }
#pragma unroll
            for (int j = 0; j < K - 1; ++j) dp[j] = dp[j + 1];
        }
#pragma unroll
        for (int j = 0; j < K - 1; ++j) x[j] = x[U + j];
    }
}

// One row of partial sums per workgroup: part[unit][(K + 1) D]; the strips' sums are added in LDS, in a fixed order.
template <typename T, int K>
__device__ __forceinline__ void conv_leave_sums(conv_shape p, const conv_sums<T, K>& sums, unsigned c, unsigned valid, unsigned unit, typename acc_of<T>::type* part)
{
    typedef typename acc_of<T>::type A;
    constexpr int V = conv_vec<T>::N;
    __shared__ A lds[256][V + 1];
    const unsigned across = 1u << p.ct_log2;
#pragma unroll
    for (int j = 0; j <= K; ++j) {
        __syncthreads();
#pragma unroll
        for (int v = 0; v < V; ++v) lds[threadIdx.x][v] = j < K ? sums.dw[j < K ? j : 0][v] : sums.db[v];
        sum_strips(lds, across, V);
        if (threadIdx.x >= across) continue;
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (v < (int)valid) part[((size_t)unit * (K + 1) + j) * p.D + c + v] = lds[threadIdx.x][v];
    }
}

template <typename T, int K, bool EXACT>
__global__ __launch_bounds__(256) void k_conv_bprop(conv_shape p, size_t lddz, unsigned items, const T* __restrict__ X, const typename acc_of<T>::type* __restrict__ W,
                                                    const typename acc_of<T>::type* __restrict__ bias, const uint32_t* __restrict__ regions,
                                                    const uint32_t* __restrict__ marks, const T* __restrict__ dZ, T* __restrict__ dX,
                                                    typename acc_of<T>::type* __restrict__ part)
{
    constexpr int V = conv_vec<T>::N;
    const unsigned x = threadIdx.x & ((1u << p.ct_log2) - 1u), y = threadIdx.x >> p.ct_log2, strips = 256u >> p.ct_log2;
    const unsigned c = ((blockIdx.y << p.ct_log2) + x) * V, valid = c < p.D ? p.D - c : 0u;
    conv_weights<T, K> w;
    conv_sums<T, K> sums;
    w.load(W, bias, p.D, c, valid);
    sums.clear();
    for (unsigned i = blockIdx.x; i < items; i += gridDim.x) {
        conv_item s;
        if (!conv_item_at(p, regions, marks, i, s)) continue;
        const unsigned strip = (s.len + strips - 1) / strips;
        conv_strip_bprop<T, K, EXACT>(p, lddz, w, sums, X, dZ, dX, c, valid, s.g, s.from + min(y * strip, s.len), s.from + min((y + 1) * strip, s.len));
    }
    conv_leave_sums<T, K>(p, sums, c, valid, blockIdx.x, part);
}

// One new row per sequence: the state's K - 1 rows move up by one.
template <typename T, int K>
__global__ __launch_bounds__(256) void k_conv_step(conv_shape p, const T* __restrict__ X, const typename acc_of<T>::type* __restrict__ W,
                                                   const typename acc_of<T>::type* __restrict__ bias, const T* state, T* into, T* __restrict__ Z)
{
    typedef typename acc_of<T>::type A;
    constexpr int V = conv_vec<T>::N;
    const size_t vecs = (p.D + V - 1) / V, i = (size_t)blockIdx.x * 256u + threadIdx.x;
    if (i >= vecs * p.N) return;
    const size_t r = i / vecs;
    const unsigned c = (unsigned)(i - r * vecs) * V, valid = p.D - c;
    conv_weights<T, K> w;
    conv_vec<T> x[K], z;
#pragma unroll
    for (int j = 0; j < K - 1; ++j) x[j].load(state + (r * (K - 1) + j) * p.D + c, valid);
    x[K - 1].load(X + r * p.ldx + c, valid);
    w.load(W, bias, p.D, c, valid);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        A a = w.b[v];
#pragma unroll
        for (int j = 0; j < K; ++j) a = fma(w.w[j][v], x[j].v[v], a);
        z.v[v] = p.silu ? a * sigmoid_of(a) : a;
    }
    z.store(Z + r * p.ldz + c, valid);
#pragma unroll
    for (int j = 0; j < K - 1; ++j) x[j + 1].store(into + (r * (K - 1) + j) * p.D + c, valid);
}

namespace {

constexpr unsigned CONV_STRIP = 32;              // rows per lane of a full segment: the K - 1 rows read again are a tenth, from the caches
constexpr size_t CONV_UNITS = 2048;              // workgroups that add up weight gradients, per tile of channels: eight per CU

size_t conv_width(int dtype) { return dtype == DBK_F64 ? 2 : 4; }

struct conv_plan { unsigned ct_log2, tiles, seg, slots, units; };

conv_plan plan_conv(int dtype, size_t N, size_t D, size_t P)
{
    conv_plan p;
    const size_t vecs = (D + conv_width(dtype) - 1) / conv_width(dtype);
    p.ct_log2 = 0;
    while (p.ct_log2 < 6 && (size_t(1) << p.ct_log2) < vecs) ++p.ct_log2;
    p.tiles = divup(vecs, size_t(1) << p.ct_log2);
    p.seg = (256u >> p.ct_log2) * CONV_STRIP;
    const size_t cap = CONV_UNITS / p.tiles ? CONV_UNITS / p.tiles : 1;
    p.slots = N > p.seg ? (unsigned)segment_slots(N, p.seg) : 0u;
    p.units = (unsigned)(P + p.slots < cap ? P + p.slots : cap);
    return p;
}

// taps, and whether rows are whole vectors
template <typename F> void with_taps(size_t K, bool exact, F f)
{
    auto g = [&](auto k) {
        if (exact) f(k, std::true_type());
        else f(k, std::false_type());
    };
    if (K == 1) g(std::integral_constant<int, 1>());
    else if (K == 2) g(std::integral_constant<int, 2>());
    else if (K == 3) g(std::integral_constant<int, 3>());
    else g(std::integral_constant<int, 4>());
}

int check_conv(int dtype, const void* X, size_t ldx, const void* W, size_t taps, size_t N, size_t D, size_t nregion, const void* Z, size_t ldz)
{
    DBK_ROW_DTYPE_OK(dtype);
    DBK_CHECK(taps >= 1 && taps <= 4, "NotImplementedError: filters of 1 to 4 taps, got %zu", taps);
    DBK_CHECK(N < (size_t(1) << 32) - 64 && D < (size_t(1) << 31) && nregion < (size_t(1) << 31), "ValueError: map too large (%zu rows, %zu channels, %zu regions)", N, D, nregion);
    DBK_CHECK(D <= size_t(65535) * 64 * 2, "ValueError: too many channels (%zu)", D);
    DBK_CHECK(nregion + N < (size_t(1) << 32) - 1, "ValueError: map too large (%zu rows, %zu regions)", N, nregion);
    DBK_CHECK(!N || !D || (X && W && Z), "ValueError: null matrix");
    DBK_CHECK(N <= 1 || (ldx >= D && ldz >= D), "ValueError: row strides must be at least the number of channels");
    return 0;
}

}  // namespace
}  // namespace dbk

using namespace dbk;

extern "C" {

int dbk_causalconv_workspace(int dtype, size_t taps, size_t N, size_t D, size_t nregion, int backward, size_t* work_bytes)
{
    DBK_ROW_DTYPE_OK(dtype);
    DBK_CHECK(work_bytes, "ValueError: null result");
    *work_bytes = 0;
    if (N && D && nregion) {
        const conv_plan p = plan_conv(dtype, N, D, nregion);
        *work_bytes = ((size_t)p.slots * 4 + 15) / 16 * 16 + (backward ? (size_t)p.units * (taps + 1) * D * acc_size(dtype) : 0);
    }
    clear_error();
    return 0;
}

int dbk_causalconv(dbk_stream_t stream, int dtype, const void* X, size_t ldx, const void* W, const void* bias, size_t taps, size_t N, size_t D,
                   const uint32_t* regions, size_t nregion, int silu, const void* state, void* Z, size_t ldz, void* last, void* work, size_t work_bytes)
{
    if (int rc = check_conv(dtype, X, ldx, W, taps, N, D, nregion, Z, ldz)) return rc;
    DBK_CHECK(!nregion || regions, "ValueError: null regions");
    if (!D || !nregion) { clear_error(); return 0; }
    const conv_plan p = plan_conv(dtype, N, D, nregion);
    DBK_CHECK(grid_fits(nregion + p.slots, 256, p.tiles), "ValueError: map too large (%zu rows, %zu regions)", N, nregion);
    DBK_CHECK(!p.slots || (work && work_bytes >= (size_t)p.slots * 4), "ValueError: the workspace has %zu bytes, %zu are needed", work_bytes, (size_t)p.slots * 4);
    const conv_shape s = {(unsigned)N, (unsigned)D, (unsigned)nregion, p.seg, p.ct_log2, (unsigned)(silu != 0), ldx, ldz};
    hipStream_t st = as_stream(stream);
    if (p.slots) k_conv_mark<<<divup(nregion, 4), 256, 0, st>>>(s, regions, (uint32_t*)work);
    with_row_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        typedef typename acc_of<T>::type A;
        with_taps(taps, D % conv_width(dtype) == 0, [&](auto k, auto exact) {
            k_conv_fprop<T, k.value, exact.value><<<dim3((unsigned)nregion + p.slots, p.tiles), 256, 0, st>>>(s, (const T*)X, (const A*)W, (const A*)bias, regions, (const uint32_t*)work,
                                                                                                        (const T*)state, (T*)Z, (T*)last);
        });
    });
    DBK_LAUNCH_OK();
}

int dbk_causalconv_bprop(dbk_stream_t stream, int dtype, const void* X, size_t ldx, const void* W, const void* bias, size_t taps, size_t N, size_t D,
                         const uint32_t* regions, size_t nregion, int silu, const void* dZ, size_t lddz, void* dX, size_t lddx, void* dW, void* dbias,
                         void* work, size_t work_bytes)
{
    if (int rc = check_conv(dtype, X, ldx, W, taps, N, D, nregion, dX, lddx)) return rc;
    DBK_CHECK(!nregion || regions, "ValueError: null regions");
    DBK_CHECK(!D || (dW && (!N || dZ)), "ValueError: null matrix");
    DBK_CHECK(N <= 1 || lddz >= D, "ValueError: row strides must be at least the number of channels");
    if (!D) { clear_error(); return 0; }
    hipStream_t st = as_stream(stream);
    if (!nregion || !N) {
        sum_partials(st, dtype, nullptr, 0, taps * D, dW, D, dbias, 0, nullptr);      // (sums of no rows: zeros)
        DBK_LAUNCH_OK();
    }
    size_t need = 0;
    if (int rc = dbk_causalconv_workspace(dtype, taps, N, D, nregion, 1, &need)) return rc;
    DBK_CHECK(work && work_bytes >= need, "ValueError: the workspace has %zu bytes, %zu are needed", work_bytes, need);
    const conv_plan p = plan_conv(dtype, N, D, nregion);
    DBK_CHECK(grid_fits(nregion + p.slots, 256, p.tiles), "ValueError: map too large (%zu rows, %zu regions)", N, nregion);
    const conv_shape s = {(unsigned)N, (unsigned)D, (unsigned)nregion, p.seg, p.ct_log2, (unsigned)(silu != 0), ldx, lddx};
    if (p.slots) k_conv_mark<<<divup(nregion, 4), 256, 0, st>>>(s, regions, (uint32_t*)work);
    void* part = (char*)work + ((size_t)p.slots * 4 + 15) / 16 * 16;
    with_row_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        typedef typename acc_of<T>::type A;
        with_taps(taps, D % conv_width(dtype) == 0, [&](auto k, auto exact) {
            k_conv_bprop<T, k.value, exact.value><<<dim3(p.units, p.tiles), 256, 0, st>>>(s, lddz, (unsigned)nregion + p.slots, (const T*)X, (const A*)W, (const A*)bias, regions,
                                                                                    (const uint32_t*)work, (const T*)dZ, (T*)dX, (A*)part);
        });
    });
    sum_partials(st, dtype, part, p.units, taps * D, dW, D, dbias, 0, nullptr);
    DBK_LAUNCH_OK();
}

int dbk_causalconv_step(dbk_stream_t stream, int dtype, const void* X, size_t ldx, const void* W, const void* bias, size_t taps, size_t n, size_t D, int silu,
                        const void* state, void* into, void* Z, size_t ldz)
{
    if (int rc = check_conv(dtype, X, ldx, W, taps, n, D, n, Z, ldz)) return rc;
    DBK_CHECK(!n || !D || taps == 1 || (state && into), "ValueError: null state");
    if (!n || !D) { clear_error(); return 0; }
    const conv_shape s = {(unsigned)n, (unsigned)D, (unsigned)n, 0u, 0u, (unsigned)(silu != 0), ldx, ldz};
    const size_t vecs = (D + conv_width(dtype) - 1) / conv_width(dtype);
    DBK_CHECK(grid_fits((n * vecs + 255) / 256, 256), "ValueError: too many sequences (%zu of %zu channels)", n, D);
    hipStream_t st = as_stream(stream);
    with_row_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        typedef typename acc_of<T>::type A;
        with_taps(taps, D % conv_width(dtype) == 0, [&](auto k, auto exact) {
            (void)exact;
            k_conv_step<T, k.value><<<divup(n * vecs, 256), 256, 0, st>>>(s, (const T*)X, (const A*)W, (const A*)bias, (const T*)state, (T*)into, (T*)Z);
        });
    });
    DBK_LAUNCH_OK();
}

}  // extern "C"
