// Shared by the operators on the rows of a map (layer norm, causal convolution, state scan): element types, vectors of
// 16 bytes of any alignment, the rows of a region, and the ordered sum of the workgroups' partial results.
#pragma once
#include "dbk_common.h"

namespace dbk {

// What one launch can hold: fewer than 2^32 threads along x (a launch of more runs without an error, and only what is over a multiple of
// 2^32 of them: 2^24 + 64 workgroups of 256 gave 64), 65535 workgroups along y and z.
inline bool grid_fits(size_t x, size_t threads, size_t y = 1, size_t z = 1) { return x < (size_t(1) << 32) / threads && y <= 65535u && z <= 65535u; }

// Rows are kept as float, double or bfloat16; every sum, statistic and state is float (double for double rows).
typedef __bf16 bf16_t;
template <typename T> struct acc_of { typedef float type; };
template <> struct acc_of<double> { typedef double type; };

inline bool row_dtype_ok(int dtype) { return dtype == DBK_F32 || dtype == DBK_F64 || dtype == DBK_BF16; }
inline size_t row_size(int dtype) { return dtype == DBK_F64 ? 8 : dtype == DBK_BF16 ? 2 : 4; }
inline size_t acc_size(int dtype) { return dtype == DBK_F64 ? 8 : 4; }

#define DBK_ROW_DTYPE_OK(dtype) \
    DBK_CHECK(dbk::row_dtype_ok(dtype), "TypeError: dtype must be DBK_F32, DBK_F64 or DBK_BF16, got %d", (int)(dtype))

// calls f(T()) for the type `dtype` names
template <typename F> inline void with_row_type(int dtype, F f)
{
    if (dtype == DBK_F32) f(float());
    else if (dtype == DBK_F64) f(double());
    else f(bf16_t());
}

// 16 bytes of T (W elements) in the accumulation type. Global memory takes vector accesses at any element's address, so odd row
// strides and odd widths use the same code as aligned ones; only a row's last, incomplete vector goes element by element.
template <typename T, int W = 16 / sizeof(T)> struct row_vec {
    static constexpr int N = W;
    typedef typename acc_of<T>::type A;
    typedef T raw __attribute__((ext_vector_type(W), aligned(sizeof(T))));
    A v[N];
    __device__ __forceinline__ void load(const T* p, unsigned valid)
    {
        if (valid >= (unsigned)N) {
            const raw r = *reinterpret_cast<const raw*>(p);
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = (A)r[i];
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = i < (int)valid ? (A)p[i] : A(0);
        }
    }
    __device__ __forceinline__ void store(T* p, unsigned valid) const
    {
        if (valid >= (unsigned)N) {
            raw r;
#pragma unroll
            for (int i = 0; i < N; ++i) r[i] = (T)v[i];          // (to bfloat16: round to nearest even)
            *reinterpret_cast<raw*>(p) = r;
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) if (i < (int)valid) p[i] = (T)v[i];
        }
    }
    __device__ __forceinline__ void fill(A x)
    {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = x;
    }
};
// A vector as it lies in memory, zeros behind its `valid` elements. EXACT: rows are whole vectors, so a vector is there or not.
template <typename T, bool EXACT, int W = 16 / sizeof(T)> struct raw_vec {
    static constexpr int N = W;
    typedef typename acc_of<T>::type A;
    typename row_vec<T, W>::raw r;
    __device__ __forceinline__ void load(const T* p, unsigned valid)
    {
        if (EXACT || valid >= (unsigned)N || valid == 0) {
            if (valid) r = *reinterpret_cast<const typename row_vec<T, W>::raw*>(p);
            else
#pragma unroll
                for (int i = 0; i < N; ++i) r[i] = (T)A(0);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) r[i] = i < (int)valid ? p[i] : (T)A(0);
        }
    }
    __device__ __forceinline__ A operator[](int i) const { return (A)r[i]; }
    // (what was converted is not kept for the next time)
    __device__ __forceinline__ void forget()
    {
        if constexpr (sizeof(T) == 2) asm volatile("" : "+v"(r));
    }
};
template <bool EXACT, typename T, int W> __device__ __forceinline__ void store_vec(const row_vec<T, W>& v, T* p, unsigned valid)
{
    if (EXACT) {
        if (valid) v.store(p, W);
    } else
        v.store(p, valid);
}

// N accumulation-type values (weights) beside one vector of T
template <typename A, int N> __device__ __forceinline__ void load_weights(A (&w)[N], const A* p, unsigned valid, A other)
{
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = p && i < (int)valid ? p[i] : other;
}

// e^x by the hardware's 2^x (1 ulp there): the rounding of x * log2(e) adds |x| / 2^24 to the relative error, which is
// small against 1 / (1 + e^-x) and against what an exponent far from zero leaves of a decay.
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ double exp2_fast(double x) { return exp2(x); }
template <typename A> __device__ __forceinline__ A exp_fast(A x) { return exp2_fast(x * A(1.4426950408889634)); }
__device__ __forceinline__ float rcp_fast(float x) { return __builtin_amdgcn_rcpf(x); }
__device__ __forceinline__ double rcp_fast(double x) { return 1.0 / x; }
// 1 / (1 + e^-x)
template <typename A> __device__ __forceinline__ A sigmoid_of(A x) { return rcp_fast(A(1) + exp_fast(-x)); }

// softplus(x) = max(x, 0) + log(1 + e), e = exp(-|x|) in (0, 1]. log(1 + e) = 2 artanh(z), z = e / (2 + e) <= 1/3, by the series
// z + z^3/3 + z^5/5 + ...: keeps the relative precision of small steps, which log(1 + e) itself loses (1 + e rounds), in a dozen
// operations; the first term left out, z^17/17, is at most 2^-29.4 of z. slope: the derivative, 1 / (1 + exp(-x)), from the same e.
__device__ __forceinline__ float softplus_of(float x, float& slope)
{
    const float e = exp_fast(-fabsf(x)), z = e * rcp_fast(2.0f + e), q = z * z, r = rcp_fast(1.0f + e);
    float s = 1.0f / 15.0f;
    s = fmaf(s, q, 1.0f / 13.0f);
    s = fmaf(s, q, 1.0f / 11.0f);
    s = fmaf(s, q, 1.0f / 9.0f);
    s = fmaf(s, q, 1.0f / 7.0f);
    s = fmaf(s, q, 1.0f / 5.0f);
    s = fmaf(s, q, 1.0f / 3.0f);
    s = fmaf(s, q, 1.0f);
    slope = x >= 0.0f ? r : e * r;
    return fmaxf(x, 0.0f) + 2.0f * z * s;                       // (a NaN comes through e)
}
__device__ __forceinline__ double softplus_of(double x, double& slope)
{
    const double e = exp(-fabs(x)), r = 1.0 / (1.0 + e);
    slope = x >= 0.0 ? r : e * r;
    return fmax(x, 0.0) + log1p(e);
}

// Sums over a workgroup's strips of rows, in LDS: v[t] += v[t + 128], v[t + 64], ... down to the first `across` (a power of two) of 256 threads.
template <typename A, int N> __device__ __forceinline__ void sum_strips(A (*v)[N], unsigned across, int n)
{
    for (unsigned o = 128; o >= across; o >>= 1) {
        __syncthreads();
        if (threadIdx.x < o)
            for (int j = 0; j < n; ++j) v[threadIdx.x][j] += v[threadIdx.x + o][j];
    }
    __syncthreads();
}

// Region r's rows, bounded by the map: [start, end), empty where the table says so or lies outside. r is the same in all lanes of a wave, and
// the compiler is told that what it reads is too: addresses and branches that depend on it are then scalar.
struct row_range { unsigned start, end; };
__device__ __forceinline__ unsigned uniform(unsigned x) { return (unsigned)__builtin_amdgcn_readfirstlane((int)x); }
__device__ __forceinline__ row_range region_rows(const uint32_t* regions, size_t r, unsigned N)
{
    row_range g;
    g.start = min(uniform(regions[2 * r]), N);
    g.end = max(min(uniform(regions[2 * r + 1]), N), g.start);
    return g;
}

// Long regions are cut into segments of L rows from their own start: segment k >= 1 of a region that starts at row s has the slot
// s / L + k. Two segments never share a slot: those of one region start L rows apart, and another region's first such start lies at
// least L rows behind its own first row. The workgroup that takes segment 0 writes the region's number into the slots of the others
// (mark_segments) and the next launch's workgroups go by slot. What a slot holds is believed only where that region does have
// a segment there (slot_segment), so the marks need no clearing: any number that passes is the right one.
__device__ __forceinline__ void mark_segments(uint32_t* marks, unsigned r, row_range g, unsigned L, unsigned thread, unsigned threads)
{
    for (uint64_t k = 1 + thread; g.start + k * L < g.end; k += threads) marks[g.start / L + k] = r;
}
__device__ __forceinline__ bool slot_segment(const uint32_t* regions, unsigned nregion, unsigned N, const uint32_t* marks, unsigned slot, unsigned L,
                                             unsigned& r, row_range& g, unsigned& k)
{
    r = uniform(marks[slot]);
    if (r >= nregion) return false;
    g = region_rows(regions, r, N);
    const unsigned q = g.start / L;
    k = slot - q;
    return slot > q && g.start + (uint64_t)k * L < g.end;
}
inline size_t segment_slots(size_t N, size_t L) { return (N + L - 1) / L; }

// Ordered sum over units of part[unit][ncol]: columns [0, n0) go to out0, the next n1 to out1, the next n2 to out2 (null:
// dropped). Defined in layernorm.hip.
int sum_partials(hipStream_t st, int dtype, const void* part, size_t units, size_t n0, void* out0, size_t n1, void* out1, size_t n2, void* out2);

}  // namespace dbk
